"""Log-probabilities straight from hidden states and an LM head, against 64 bits.

Tolerances are sums of roundings: u = 2^-24 for each fp32 operation, half a step (2^-8) of
bf16 for what is rounded to it: dz once, as the matrix cores' operand, the softmax's numerators
that a forward keeps, and the gradients.
"""

import pytest
import torch
import torch.nn.functional as F

import nano_qwen_amd as nq
from nano_qwen_amd.model import ModelConfig, Qwen3Model
from tests.helpers import randn, say
from tests.test_gpu_losses import U, ragged, within

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16
HALF = 2.0 ** -8


def reference(h, w, labels, dy, T, ignore=-100):
    """(logprobs, dh, dw) and their tolerances."""
    (V, H), shape = w.shape, labels.shape
    h, labels, dy = h.double().reshape(-1, H), labels.reshape(-1), dy.double().reshape(-1)
    w = w.double()
    z = h @ w.t() / T
    size = h.abs() @ w.abs().t() / T           # sums of H products err by at most H u of their terms' sizes
    logp = torch.log_softmax(z, -1)
    keep = labels != ignore
    at = labels.clamp(0, V - 1)[:, None]
    bad = keep & ((labels < 0) | (labels >= V))
    lp = torch.where(bad, torch.nan, torch.where(keep, logp.gather(1, at)[:, 0], 0.0))
    # z off by H u of its terms; the exponent by |z - m| u, 64 terms one after the other and a
    # few tens of joins
    err = H * U * size.amax(1) + (2 * (z.amax(1) - z.amin(1)) + 200) * U
    tol = 2 * err + 4 * U * lp.abs().nan_to_num(0)
    g = torch.where(keep, dy, 0.0) / T
    g = torch.where(bad, torch.nan, g)[:, None]
    p = torch.exp(logp)
    dz = torch.where(keep[:, None], -p * g, 0.0).scatter_add(1, at, g)
    dh, dw = dz @ w, dz.t() @ h
    # |dz| off by half a step and its softmax by another, where kept, and err; fp32 sums over the terms
    off = (dz.abs() * HALF + (-p * g).abs() * HALF * 1.01 + g.abs() * p * err[:, None] * 2 + 1e-37).nan_to_num(0)
    tol_h = off @ w.abs() + V * U * (dz.abs().nan_to_num(0) @ w.abs()) + HALF * dh.abs().nan_to_num(0) + 1e-37
    tol_w = off.t() @ h.abs() + len(h) * U * (dz.abs().nan_to_num(0).t() @ h.abs()) + HALF * dw.abs().nan_to_num(0) + 1e-37
    return lp.view(shape), dh.view(*shape, H), dw, tol.view(shape), tol_h.view(*shape, H), tol_w


def run(h, w, labels, dy, T=1.0, **kw):
    hd, wd = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    lp = nq.linear_logprobs(hd, wd, labels.to(DEV), temperature=T, **kw)
    return (lp, *torch.autograd.grad(lp, (hd, wd), dy.to(DEV)))


def check(h, w, labels, dy, T=1.0, what="", **kw):
    lp, dh, dw = run(h, w, labels, dy, T, **kw)
    want = reference(h, w, labels, dy, T, kw.get("ignore_index", -100))
    assert lp.dtype == torch.float32 and lp.shape == labels.shape
    assert dh.dtype == dw.dtype == BF and dh.shape == h.shape and dw.shape == w.shape
    for name, got, ref, tol in zip(("logprobs", "dhidden", "dweight"), (lp, dh, dw), want, want[3:]):
        within(got, ref, tol, f"{what} {name}")


def inputs(shape, V, H, seed, prompt=0.0):
    h = randn(*shape, H, seed=seed).to(BF)
    w = (randn(V, H, seed=seed + 1) * 2 / H ** 0.5).to(BF)
    labels = torch.randint(0, V, shape, generator=torch.Generator().manual_seed(seed + 2))
    if prompt:
        labels[torch.rand(shape, generator=torch.Generator().manual_seed(seed + 3)) < prompt] = -100
    return h, w, labels, randn(*shape, seed=seed + 4)


# one row to several tiles of both token extents; a vocabulary of one entry, below, at and past
# tiles; widths below, at and past a step and a tile
@pytest.mark.parametrize("rows,V,H", [(1, 1, 8), (1, 300, 64), (3, 256, 72), (33, 1000, 520), (64, 513, 256), (65, 513, 264),
                                      (256, 256, 256), (257, 1025, 64), (700, 777, 328), (300, 5003, 1024), (2, 20000, 128), (90, 640, 248), (130, 1001, 256)])
def test_linear_logprobs(rows, V, H):
    say(f"linear_logprobs {rows} x {V} x {H}")
    h, w, labels, dy = inputs((rows,), V, H, 100)
    labels[rows // 2] = V - 1
    for recompute in (False, True):
        check(h, w, labels, dy, T=0.7 if V % 2 else 1.0, what=f"{rows}x{V}x{H}", recompute=recompute)


@pytest.mark.parametrize("rows,share", [(50, 0.5), (600, 0.3), (600, 0.97), (64, 1.0), (300, 1.0)])
def test_linear_logprobs_leaves_ignored_rows_out(rows, share):
    """Kept rows in any pattern; ignored ones are not read, whatever they hold."""
    say(f"linear_logprobs ignored {rows} {share}")
    h, w, labels, dy = inputs((rows,), 700, 264, 110)
    drop = torch.rand(rows, generator=torch.Generator().manual_seed(113)) < share if share < 1 else torch.ones(rows, dtype=torch.bool)
    labels[drop] = -7
    want = reference(h, w, labels, dy, 1.0, -7)
    h, dy = h.clone(), dy.clone()
    h[drop], dy[drop] = float("nan"), float("nan")
    for recompute in (False, True):
        got = run(h, w, labels, dy, ignore_index=-7, recompute=recompute)
        for name, a, ref, tol in zip(("logprobs", "dhidden", "dweight"), got, want, want[3:]):
            within(a, ref, tol, name)
        assert not got[0][drop.to(DEV)].any() and not got[1][drop.to(DEV)].any()


@pytest.mark.parametrize("rows", [40, 140])
@pytest.mark.parametrize("recompute", [False, True])
def test_linear_logprobs_special_values(rows, recompute):
    """Labels outside the vocabulary, NaN and infinite hidden states, a masked-out vocabulary entry."""
    say(f"linear_logprobs special values {rows} {recompute}")
    H = 64 if rows == 40 else 264  # nothing is kept, and the softmax's numerators
    h, w, labels, dy = inputs((rows,), 300, H, 120)
    labels[3], labels[9] = 300, -1
    lp, dh, dw = run(h, w, labels, dy, recompute=recompute)
    want = reference(h, w, labels, dy, 1.0)
    within(lp, want[0], want[3], "labels outside")
    within(dh, want[1], want[4], "labels outside, dhidden")
    assert torch.isnan(dw).all()
    labels[3], labels[9] = 0, 1
    h[5], h[6, 7] = float("nan"), float("inf")
    lp, dh, _ = run(h, w, labels, dy, recompute=recompute)
    assert torch.isnan(lp[[5, 6]]).all() and torch.isfinite(lp).sum() == rows - 2
    assert torch.isnan(dh[[5, 6]]).any(1).all() and torch.isfinite(dh).all(1).sum() == rows - 2
    # logits far apart: the others' probabilities vanish, and nothing overflows; a label almost certain
    h, w, labels, dy = inputs((rows,), 300, H, 121)
    check(h * 64, w, labels, dy, what="far apart", recompute=recompute)
    h = (w[labels].float() * 3).to(BF)
    check(h, w, labels, dy, what="certain labels", recompute=recompute)


def test_linear_logprobs_strides_and_shapes():
    say("linear_logprobs strides")
    h, w, labels, dy = inputs((3, 41), 500, 256, 130, prompt=0.2)
    big = torch.zeros(3, 42, 272, dtype=BF)
    big[:, 1:, 8:264] = h
    views = {"sliced": big.to(DEV)[:, 1:, 8:264], "misaligned": torch.cat([h[..., :1], h], -1).to(DEV)[..., 1:],
             "transposed": h.transpose(0, 1).contiguous().to(DEV).transpose(0, 1)}
    want = reference(h, w, labels, dy, 1.0)
    for name, view in views.items():
        leaf, wl = view.detach().requires_grad_(), w.t().contiguous().to(DEV).t().requires_grad_()
        lp = nq.linear_logprobs(leaf, wl, labels.to(DEV).int())
        grads = torch.autograd.grad(lp, (leaf, wl), dy.to(DEV))
        for a, ref, tol in zip((lp, *grads), want, want[3:]):
            within(a, ref, tol, name)
    # one of the gradients alone, and none
    only = nq.linear_logprobs(views["sliced"].requires_grad_(), w.to(DEV), labels.to(DEV))
    (dh,) = torch.autograd.grad(only, views["sliced"], dy.to(DEV))
    within(dh, want[1], want[4], "dhidden alone")
    wl = w.to(DEV).requires_grad_()
    (dw,) = torch.autograd.grad(nq.linear_logprobs(h.to(DEV), wl, labels.to(DEV)), wl, dy.to(DEV))
    within(dw, want[2], want[5], "dweight alone")
    assert nq.linear_logprobs(h.to(DEV), w.to(DEV), labels.to(DEV)).grad_fn is None
    one = nq.linear_logprobs(h[0, 0].to(DEV), w.to(DEV), labels[0, 0].to(DEV))
    within(one, want[0][0, 0], want[3][0, 0], "one row")
    empty, wl = h[:0].to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    lp = nq.linear_logprobs(empty, wl, labels[:0].to(DEV))
    assert lp.shape == (0, 41) and not torch.autograd.grad(lp.sum(), wl)[0].any()


@pytest.mark.parametrize("shape", [(1,), (1, 1), (3, 1), (1, 3)])
def test_linear_logprobs_of_axes_of_one(shape):
    """An axis of one has any stride, here no multiple of 16 bytes."""
    say(f"linear_logprobs axes of one {shape}")
    h, w, labels, dy = inputs(shape, 100, 64, 135)
    big = torch.zeros(2 * 2 * 4 * 8 * 73, dtype=BF, device=DEV)
    strides = [73 if n == 1 else 8 * 72 for n in shape] + [1]
    view = big.as_strided((*shape, 64), strides)
    with torch.no_grad():
        view.copy_(h)
    leaf, wl = view.detach().requires_grad_(), w.to(DEV).requires_grad_()
    lp = nq.linear_logprobs(leaf, wl, labels.to(DEV))
    got = (lp, *torch.autograd.grad(lp, (leaf, wl), dy.to(DEV)))
    want = reference(h, w, labels, dy, 1.0)
    for a, ref, tol in zip(got, want, want[3:]):
        within(a, ref, tol, "axes of one")


def test_linear_logprobs_many_rows():
    """More rows than 2048 gathering workgroups of 16 take: each counts those before its own."""
    say("linear_logprobs many rows")
    rows, V, H = 200003, 40, 8
    g = torch.Generator(device=DEV).manual_seed(145)
    h = torch.randn(rows, H, generator=g, device=DEV).to(BF).requires_grad_()
    w = torch.randn(V, H, generator=g, device=DEV).to(BF)
    labels = torch.randint(0, V, (rows,), generator=g, device=DEV)
    labels[torch.rand(rows, generator=g, device=DEV) < 0.4] = -100
    dy = torch.randn(rows, generator=g, device=DEV)
    lp = nq.linear_logprobs(h, w, labels)
    (dh,) = torch.autograd.grad(lp, h, dy)
    want = reference(h.detach(), w, labels, dy, 1.0)
    within(lp, want[0].cpu(), want[3].cpu(), "logprobs")
    within(dh, want[1].cpu(), want[4].cpu(), "dhidden")


@pytest.mark.parametrize("recompute", [False, True])
def test_linear_logprobs_several_ranges(recompute):
    """So many rows that the backward takes the vocabulary in several ranges, the last a short one."""
    say(f"linear_logprobs several ranges {recompute}")
    rows, V, H = 70000, 9001, 256
    g = torch.Generator(device=DEV).manual_seed(140)
    h = torch.randn(rows, H, generator=g, device=DEV).to(BF).requires_grad_()
    w = (torch.randn(V, H, generator=g, device=DEV) * 0.1).to(BF).requires_grad_()
    labels = torch.randint(0, V, (rows,), generator=g, device=DEV)
    labels[::3] = -100
    dy = torch.randn(rows, generator=g, device=DEV)
    lp = nq.linear_logprobs(h, w, labels, recompute=recompute)
    dh, dw = torch.autograd.grad(lp, (h, w), dy)
    # dw row by row over the kept rows of all; a sample of the rows of dh
    at = torch.arange(0, rows, 97, device=DEV)
    want = [t.cpu() for t in reference(h.detach()[at], w.detach(), labels[at], dy[at], 1.0)]
    within(lp[at], want[0], want[3], "logprobs")
    within(dh[at], want[1], want[4], "dhidden")
    total, tol = torch.zeros(V, H, dtype=torch.float64, device=DEV), torch.zeros(V, H, dtype=torch.float64, device=DEV)
    for part in torch.arange(rows, device=DEV).split(5000):
        r = reference(h.detach()[part], w.detach(), labels[part], dy[part], 1.0)
        total += r[2]
        tol += r[5] - HALF * r[2].abs()
    # the same bound over all rows: each part's terms' roundings, the sum's own, and one rounding of the result
    within(dw, total.cpu(), (tol * rows / 5000 + HALF * total.abs()).cpu(), "dweight")
    # without its bound's worst case: half a step of dz, independent from term to term, and of the result
    assert float((dw.double() - total).norm() / total.norm()) < 2 * HALF


def test_linear_logprobs_differences():
    """The gradients against central differences of the operator itself."""
    say("linear_logprobs differences")
    h, w, labels, dy = inputs((20,), 90, 64, 150)
    _, dh, dw = run(h, w, labels, dy)
    # steps along the gradients that bf16 holds: whole units in the last place of a power of two
    dh_step, dw_step = (2.0 ** -6 * torch.sign(t.float().cpu()) for t in (dh, dw))
    for what, hs, ws, along in (("hidden", dh_step, 0 * dw_step, (dh.double().cpu() * dh_step).sum()),
                                ("weight", 0 * dh_step, dw_step, (dw.double().cpu() * dw_step).sum())):
        ends = []
        for sign in (1, -1):
            a, b = (h.float() + sign * hs).to(BF), (w.float() + sign * ws).to(BF)
            ends.append((a, b, float((nq.linear_logprobs(a.to(DEV), b.to(DEV), labels.to(DEV)).double().cpu() * dy).sum())))
        # the step as bf16 took it
        real = ((dh.double().cpu() * (ends[0][0].double() - ends[1][0].double())).sum()
                + (dw.double().cpu() * (ends[0][1].double() - ends[1][1].double())).sum())
        diff = ends[0][2] - ends[1][2]
        # a step s changes a logit by at most s |.|_1 <= D; the third-order term is under D^3 per row
        D = 2.0 ** -6 * float((w.abs().sum(1).max() if what == "hidden" else h.abs().sum(1).max()))
        assert abs(diff - float(real)) <= 2 * D ** 3 * float(dy.abs().sum()) + 2 * HALF * float(
            (dh.double().cpu().abs() * dh_step.abs()).sum() + (dw.double().cpu().abs() * dw_step.abs()).sum()), what


def test_linear_logprobs_refusals():
    h, w, y = torch.zeros(4, 16, device=DEV, dtype=BF), torch.zeros(9, 16, device=DEV, dtype=BF), torch.zeros(4, dtype=torch.long, device=DEV)
    for err, args in ((RuntimeError, (h.cpu(), w, y)), (RuntimeError, (h, w.cpu(), y)), (RuntimeError, (h, w, y.cpu())),
                      (TypeError, (h.float(), w, y)), (TypeError, (h, w.float(), y)), (TypeError, (h, w, y.float())),
                      (ValueError, (h[:, :8], w, y)), (ValueError, (h[:, :12], w[:, :12], y)), (ValueError, (h, w[:0], y)),
                      (ValueError, (h, w, y[:3])), (ValueError, (h, w[0], y)), (ValueError, (h[:, :0], w[:, :0], y))):
        with pytest.raises(err):
            nq.linear_logprobs(*args)
    with pytest.raises(ValueError, match="temperature"):
        nq.linear_logprobs(h, w, y, temperature=0.0)
    with pytest.raises(RuntimeError):
        hg = h.clone().requires_grad_()
        (d,) = torch.autograd.grad(nq.linear_logprobs(hg, w, y).sum(), hg, create_graph=True)
        torch.autograd.grad(d.sum(), hg)


def test_linear_logprobs_bits_streams_graph():
    """The same bits on any stream and in a replayed graph."""
    say("linear_logprobs streams and graph")
    h, w, labels, dy = inputs((5, 77), 3001, 256, 160, prompt=0.3)
    hd, wd, yd, gd = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_(), labels.to(DEV), dy.to(DEV)

    def step():
        lp = nq.linear_logprobs(hd, wd, yd)
        grads = torch.autograd.grad(lp, (hd, wd), gd)
        return [lp.detach(), *grads]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(3):
        with torch.no_grad():
            hd.copy_(randn(5, 77, 256, seed=170 + i).to(BF))
            yd.copy_(torch.randint(0, 3001, (5, 77), generator=torch.Generator().manual_seed(180 + i)))
            yd[:, :20 * i] = -100
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        want = step()
        streams = [torch.cuda.Stream() for _ in range(2)]
        more = []
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                more.append(step())
        torch.cuda.synchronize()
        for other in (got, *more):
            assert all(torch.equal(a, b) for a, b in zip(other, want)), i


def small_model(dtype):
    cfg = ModelConfig(vocab_size=997, hidden_size=64, intermediate_size=128, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, head_dim=32)
    torch.manual_seed(3)
    return Qwen3Model(cfg).to(DEV, dtype)


@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_model_token_logprobs(dtype):
    """A model's own log-probabilities are those of its logits, shifted as its loss is."""
    say(f"model token_logprobs {dtype}")
    model = small_model(dtype)
    ids = torch.randint(0, 997, (3, 21), generator=torch.Generator().manual_seed(4)).to(DEV)
    labels = ids.clone()
    labels[:, :5] = -100
    lp = model.token_logprobs(ids, labels)
    out = model(ids, labels=labels)
    assert lp.shape == (3, 20)
    # from the model's hidden states in 64 bits
    z = out["hidden_states"][:, :-1].double() @ model.lm_head.weight.double().t()
    want = torch.log_softmax(z, -1).gather(-1, ids[:, 1:, None])[..., 0]
    want = torch.where(labels[:, 1:] != -100, want, 0.0)
    within(lp, want.cpu(), 1e-4, "logprobs")  # 64 products and 997 exponentials of fp32, values under 10
    within(model.token_logprobs(ids)[:, 5:], want[:, 5:].cpu(), 1e-4, "labels by default")
    grads = torch.autograd.grad(-lp.sum() / (labels[:, 1:] != -100).sum(), list(model.parameters()))
    wants = torch.autograd.grad(out["loss"].float(), list(model.parameters()))
    for (name, _), a, b in zip(model.named_parameters(), grads, wants):
        # bf16: the loss's own path rounds logits, their gradient and each layer's to 2^-8 a piece
        lim = 0.05 if dtype == BF else 1e-4
        assert float((a.double() - b.double()).norm() / b.double().norm().clamp(min=1e-30)) < lim, name


def test_model_token_logprobs_runs_what_stands_in_its_head():
    """A hooked or replaced LM head runs as it is."""
    say("model token_logprobs of a changed head")
    model = small_model(BF)
    ids = torch.randint(0, 997, (2, 9), generator=torch.Generator().manual_seed(8)).to(DEV)
    with torch.no_grad():
        plain = model.token_logprobs(ids)
        handle = model.lm_head.register_forward_hook(lambda mod, args, out: out * 0.5)
        halved = model.token_logprobs(ids)
        handle.remove()
        want = torch.log_softmax((model(ids)["logits"][:, :-1] * 0.5).double(), -1).gather(-1, ids[:, 1:, None])[..., 0]
        within(halved, want.cpu(), 1e-4, "hooked head")
        assert torch.equal(model.token_logprobs(ids), plain)
        model.lm_head = torch.nn.Sequential(model.lm_head, torch.nn.Identity())
        z = model(ids)["logits"][:, :-1].double()
        want = torch.log_softmax(z, -1).gather(-1, ids[:, 1:, None])[..., 0]
        within(model.token_logprobs(ids), want.cpu(), 1e-4, "replaced head")
        assert model.token_logprobs(ids[:, :1]).shape == (2, 0)


def test_preference_and_policy_steps_of_a_model():
    """The operators together as a preference step and a policy step run them, against 64-bit losses over the
    same log-probabilities; what the optimizer sees has a gradient for every parameter."""
    say("preference and policy steps")
    model, ref = small_model(BF), small_model(BF)
    with torch.no_grad():
        for p in ref.parameters():
            p.add_(0.01 * torch.randn(p.shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(p.numel())).to(BF))
    g = torch.Generator().manual_seed(5)
    ids = torch.randint(0, 997, (8, 33), generator=g).to(DEV)
    keep = ragged(8, 33, 6)
    keep[4] = True
    keep[:, :6] = False
    labels = torch.where(keep.to(DEV), ids, -100)
    mask = (labels != -100)[:, 1:]
    lp = model.token_logprobs(ids, labels)
    with torch.no_grad():
        rlp = ref.token_logprobs(ids, labels)
    loss, wc, wr = nq.preference_loss(lp[:4], lp[4:], rlp[:4], rlp[4:], chosen_mask=mask[:4], rejected_mask=mask[4:], beta=0.5)
    d = (lp.double() - rlp).sum(1)
    want = -F.logsigmoid(0.5 * (d[:4] - d[4:])).mean()
    assert abs(float(loss.detach()) - float(want.detach())) < 1e-6
    adv = torch.linspace(-1, 1, 8, device=DEV)
    pol, kl, _ = nq.policy_loss(lp, lp.detach() + 0.05, adv, ref_logprobs=rlp, mask=mask, kl_coef=0.1, reduction="sequence")
    params = list(model.parameters())
    got = torch.autograd.grad(loss + pol, params, retain_graph=True)
    q = rlp.double() - lp.double()
    r = torch.exp(lp.double() - (lp.detach() + 0.05))
    each = -torch.minimum(r * adv[:, None], r.clamp(0.8, 1.2) * adv[:, None]) + 0.1 * (torch.expm1(q) - q)
    ref_pol = ((each * mask).sum(1) / mask.sum(1).clamp(min=1)).mean()
    want = torch.autograd.grad(want + ref_pol, params)
    for a, b, (name, _) in zip(got, want, model.named_parameters()):
        # the two gradients of the log-probabilities differ by some u: the same bf16 backward follows
        assert torch.isfinite(a).all() and float((a.double() - b.double()).norm()) <= 0.01 * float(b.double().norm()) + 1e-12, name
    # under gradient checkpointing, whose saved tensors are made anew in the backward, the same bits
    model.gradient_checkpointing = True
    model.train()
    lp2 = model.token_logprobs(ids, labels)
    assert torch.equal(lp2, lp)
    loss2, *_ = nq.preference_loss(lp2[:4], lp2[4:], rlp[:4], rlp[4:], chosen_mask=mask[:4], rejected_mask=mask[4:], beta=0.5)
    pol2, *_ = nq.policy_loss(lp2, lp.detach() + 0.05, adv, ref_logprobs=rlp, mask=mask, kl_coef=0.1, reduction="sequence")
    for a, b in zip(torch.autograd.grad(loss2 + pol2, params), got):
        assert torch.equal(a, b)


def test_model_token_logprobs_runs_a_patched_head():
    """What offloading and adapter code puts on the head's instance, and hooks of all modules, run."""
    say("model token_logprobs of a patched head")
    model = small_model(BF)
    ids = torch.randint(0, 997, (2, 9), generator=torch.Generator().manual_seed(9)).to(DEV)
    head = model.lm_head
    inner = head.forward
    with torch.no_grad():
        plain = model.token_logprobs(ids)
        head.forward = lambda x: inner(x) * 0.5
        want = torch.log_softmax(model(ids)["logits"][:, :-1].double(), -1).gather(-1, ids[:, 1:, None])[..., 0]
        within(model.token_logprobs(ids), want.cpu(), 1e-4, "patched forward")
        del head.forward
        handle = torch.nn.modules.module.register_module_forward_hook(
            lambda mod, args, out: out * 0.5 if mod is head else None)
        try:
            within(model.token_logprobs(ids), want.cpu(), 1e-4, "global hook")
        finally:
            handle.remove()
        assert torch.equal(model.token_logprobs(ids), plain)


def test_model_token_logprobs_memory():
    """What a call holds until its backward: two bytes a token and vocabulary entry, none with recompute."""
    say("model token_logprobs memory")
    cfg = ModelConfig(vocab_size=20000, hidden_size=256, intermediate_size=256, num_hidden_layers=1, num_attention_heads=4,
                      num_key_value_heads=2, head_dim=64)
    torch.manual_seed(3)
    model = Qwen3Model(cfg).to(DEV, BF)
    ids = torch.randint(0, 20000, (2, 501), generator=torch.Generator().manual_seed(10)).to(DEV)
    held, grads, outs = [], [], []
    for recompute in (False, True):
        for _ in range(2):  # the second without the first call's lasting allocations
            torch.cuda.synchronize()
            before = torch.cuda.memory_allocated()
            lp = model.token_logprobs(ids, recompute=recompute)
            held.append(torch.cuda.memory_allocated() - before)
            g = torch.autograd.grad(lp.sum(), model.lm_head.weight)[0]
            outs.append(lp.detach())
            del lp
        grads.append(g)
    logits = 2 * 1000 * 20000
    assert held[1] - held[3] > 0.99 * logits and held[3] < 0.5 * logits
    assert torch.equal(outs[1], outs[3])
    # numerators rounded to bf16 once more: half a step of each
    assert float((grads[0].double() - grads[1].double()).norm() / grads[1].double().norm()) < 2 * HALF


# At most 64 rows: 768 workgroups of 128 entries each, which take a second tile from 98305 entries on;
# weights of more than 256 MB are loaded past the cache.
@pytest.mark.parametrize("rows,V,H", [(64, 100003, 64), (33, 151936, 8), (1, 131500, 1024), (33, 131500, 1024), (64, 151936, 1024)])
def test_linear_logprobs_few_rows_of_many_tiles(rows, V, H):
    say(f"linear_logprobs few rows {rows} x {V} x {H}")
    g = torch.Generator(device=DEV).manual_seed(190)
    h = torch.randn(rows, H, generator=g, device=DEV).to(BF).requires_grad_()
    w = (torch.randn(V, H, generator=g, device=DEV) * 2 / H ** 0.5).to(BF).requires_grad_()
    labels = torch.randint(0, V, (rows,), generator=g, device=DEV)
    dy = torch.randn(rows, generator=g, device=DEV)
    # tiles go to the 8 XCDs in runs, 96 of a run at first and the others second: a label in each run's last tiles
    per = (-(-V // 128) + 7) // 8
    assert per > 96
    for i in range(min(rows, 16)):
        labels[-1 - i] = min(((i % 8) * per + 96 + i // 8) * 128 + 5 * i, V - 1)
    if rows > 1:
        labels[0], labels[1:rows // 2:3] = V - 1, -100
    lp = nq.linear_logprobs(h, w, labels)
    dh, dw = torch.autograd.grad(lp, (h, w), dy)
    want = reference(h.detach(), w.detach(), labels, dy, 1.0)
    with torch.no_grad():
        assert torch.equal(nq.linear_logprobs(h, w, labels), lp)
    for name, got, ref, tol in zip(("logprobs", "dhidden"), (lp, dh), want, want[3:]):
        within(got, ref.cpu(), tol.cpu(), name)
    bad = (dw.double() - want[2]).abs() > want[5]
    assert not bool(bad.any()) and bool(torch.isfinite(dw).all()), "dweight"


def test_model_token_logprobs_under_autocast():
    """fp32 weights under bf16 autocast: the head's logits are bf16, and the log-probabilities are theirs."""
    say("model token_logprobs under autocast")
    model = small_model(torch.float32)
    ids = torch.randint(0, 997, (3, 21), generator=torch.Generator().manual_seed(11)).to(DEV)
    with torch.autocast("cuda", torch.bfloat16):
        lp = model.token_logprobs(ids)
        z = model.lm_head(model(ids)["hidden_states"][:, :-1])
    assert z.dtype == BF and lp.dtype == torch.float32
    want = torch.log_softmax(z.double(), -1).gather(-1, ids[:, 1:, None])[..., 0]
    within(lp, want.detach().cpu(), 1e-4, "logprobs")  # 997 exponentials of fp32, values under 10
    grads = torch.autograd.grad(-lp.mean(), list(model.parameters()))
    with torch.autocast("cuda", torch.bfloat16):
        loss = model(ids, labels=ids)["loss"]
    wants = torch.autograd.grad(loss.float(), list(model.parameters()))
    for (name, _), a, b in zip(model.named_parameters(), grads, wants):
        # logits, their gradient and each layer's rounded to 2^-8 a piece in both
        assert a.dtype == torch.float32 and float((a.double() - b.double()).norm() / b.double().norm().clamp(min=1e-30)) < 0.05, name
