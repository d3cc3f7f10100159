"""The LM head's gradients against central differences of the operator, along directions that are fixed
before any gradient is computed; what the check would let pass is measured on the CPU.

The logits move by exactly t u along a step of hidden states or of weights (both steps are exact in
bf16).  A row's log-probability then has a third derivative of at most R^3 / (6 sqrt 3), R the range of
u over the vocabulary: the third central moment of a variable within an interval.
"""

import math

import pytest
import torch

import nano_qwen_amd as nq
from tests.helpers import say
from tests.test_gpu_head import reference

BF = torch.bfloat16
STEP = 2.0 ** -7
SIZES = [(20, 90, 64), (64, 700, 64), (70, 300, 256)]  # few rows; as many as those; rows whose numerators are kept


def case(rows, V, H):
    """Operands on coarse grids, steps that bf16 adds exactly, labels among the first entries, whose weights
    lie above the others': hidden states alternate in sign, so the logits stay near 0 all the same."""
    g = torch.Generator().manual_seed(200 + rows)
    sign = torch.where(torch.arange(H) % 2 == 0, 1.0, -1.0)
    first = torch.where(torch.arange(V) < 10, 1.0, -1.0)
    h = sign * 0.5 + torch.randint(-3, 4, (rows, H), generator=g) / 16
    w = first[:, None] * 0.25 + torch.randint(-4, 5, (V, H), generator=g) / 32
    labels = torch.randint(0, 10, (rows,), generator=g)
    dy = 0.5 + torch.rand(rows, generator=g)
    stepped = (torch.arange(H) < 64).float()  # 64 of the width move, so that R stays small
    steps = {"hidden": (STEP * stepped.expand(rows, H), torch.zeros(V, H)),
             "weight": (torch.zeros(rows, H), STEP * first[:, None] * sign * stepped)}
    for t, s in ((h, steps["hidden"][0]), (w, steps["weight"][1])):
        for u in (t, t + s, t - s):
            assert torch.equal(u.to(BF).float(), u)
    return h, w, labels, dy, steps


def bound(h, w, labels, dy, hs, ws):
    """How far f(1) - f(-1) may be from twice the gradients along the step."""
    u = hs.double() @ w.double().t() + h.double() @ ws.double().t()
    R = u.amax(1) - u.amin(1)
    third = float((dy.double() * R ** 3).sum()) / (6 * math.sqrt(3)) / 3
    tol = 0.0
    for sign in (1, -1):
        tol += float((dy * reference(h + sign * hs, w + sign * ws, labels, dy, 1.0)[3]).sum())
    _, _, _, _, th, tw = reference(h, w, labels, dy, 1.0)
    return third + tol + 2 * float((hs.abs() * th).sum() + (ws.abs() * tw).sum())


def along(dh, dw, hs, ws):
    return 2 * float((dh.double().cpu() * hs).sum() + (dw.double().cpu() * ws).sum())


@pytest.mark.parametrize("rows,V,H", SIZES)
@pytest.mark.parametrize("what", ["hidden", "weight"])
def test_differences_tell_wrong_gradients(rows, V, H, what):
    """In 64 bits: the formula's gradients pass, and the same halved, without the softmax's term, with half
    of it or without the label's do not, by a wide margin."""
    h, w, labels, dy, steps = case(rows, V, H)
    hs, ws = steps[what]
    ends = [float((reference(h + s * hs, w + s * ws, labels, dy, 1.0)[0] * dy).sum()) for s in (1, -1)]
    lim = bound(h, w, labels, dy, hs, ws)
    _, dh, dw, *_ = reference(h, w, labels, dy, 1.0)
    diff = ends[0] - ends[1]
    assert abs(diff - along(dh, dw, hs, ws)) <= lim < 0.05 * abs(diff)
    hot = torch.nn.functional.one_hot(labels, V).double() * dy.double()[:, None]
    oh, ow = hot @ w.double(), hot.t() @ h.double()
    for name, gh, gw in (("half", dh / 2, dw / 2), ("no softmax", oh, ow), ("no label", dh - oh, dw - ow),
                         ("half the softmax", (dh + oh) / 2, (dw + ow) / 2)):
        assert abs(diff - along(gh, gw, hs, ws)) > 4 * lim, name


@pytest.mark.gpu
@pytest.mark.parametrize("rows,V,H", SIZES)
@pytest.mark.parametrize("what", ["hidden", "weight"])
@pytest.mark.parametrize("recompute", [False, True])
def test_linear_logprobs_differences_along_fixed_steps(rows, V, H, what, recompute):
    say(f"linear_logprobs differences {rows} x {V} x {H} {what} {recompute}")
    h, w, labels, dy, steps = case(rows, V, H)
    hs, ws = steps[what]
    leaves = [t.to(BF).cuda().requires_grad_() for t in (h, w)]
    lp = nq.linear_logprobs(*leaves, labels.cuda(), recompute=recompute)
    dh, dw = torch.autograd.grad(lp, leaves, dy.cuda())
    ends = [nq.linear_logprobs((h + s * hs).to(BF).cuda(), (w + s * ws).to(BF).cuda(), labels.cuda()) for s in (1, -1)]
    diff = float(((ends[0].double() - ends[1].double()).cpu() * dy).sum())
    assert abs(diff - along(dh, dw, hs, ws)) <= bound(h, w, labels, dy, hs, ws)
