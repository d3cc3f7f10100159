"""The loss operators' checks that need no GPU: what the C entry points refuse before any launch, the
workspaces they ask for, and that host tensors raise."""

import ctypes

import pytest
import torch

import nano_qwen_amd as nq
from nano_qwen_amd import _lib

P = ctypes.c_void_p(1 << 20)       # never dereferenced: every call below is refused before a launch
ODD = ctypes.c_void_p((1 << 20) + 1)
BF, F32 = _lib.NQ_DTYPE_BF16, _lib.NQ_DTYPE_F32
INV, UNS, WS = _lib.NQ_ERR_INVALID, _lib.NQ_ERR_UNSUPPORTED, _lib.NQ_ERR_WORKSPACE
BIG = 1 << 62


def refused(fn, want, match, *args):
    lib = _lib.load()
    rc = getattr(lib, fn)(*args)
    assert rc == want, (fn, rc, lib.nq_last_error())
    assert match.encode() in lib.nq_last_error(), lib.nq_last_error()


def tokens(x=P, bs=0, rs=100, labels=P, out=P, stats=P, ws=P, n=BIG, B=1, S=4, V=100, dt=BF, T=1.0):
    return (x, bs, rs, labels, out, stats, ws, n, B, S, V, dt, T, -100, None)


def tokens_bwd(x=P, bs=0, rs=100, labels=P, stats=P, dy=P, dx=P, B=1, S=4, V=100, dt=BF, T=1.0):
    return (x, bs, rs, labels, stats, dy, dx, B, S, V, dt, T, -100, None)


def head(x=P, bs=0, rs=64, w=P, labels=P, out=P, stats=P, kept=None, nk=0, ws=P, n=BIG, B=1, S=4, V=100, H=64, T=1.0):
    return (x, bs, rs, w, labels, out, stats, kept, nk, ws, n, B, S, V, H, T, -100, None)


def head_bwd(x=P, bs=0, rs=64, w=P, labels=P, stats=P, kept=None, nk=0, dy=P, dh=P, dw=P, ws=P, n=BIG, B=1, S=4, V=100, H=64,
             T=1.0):
    return (x, bs, rs, w, labels, stats, kept, nk, dy, dh, dw, ws, n, B, S, V, H, T, -100, None)


def preference(c=P, r=P, loss=P, wc=P, wr=P, coef=P, ws=P, n=BIG, B=20, Sc=9, Sr=9, kind=0, beta=0.1, e=0.0):
    return (c, 9, r, 9, None, 0, None, 0, None, 0, None, 0, loss, wc, wr, coef, ws, n, B, Sc, Sr, kind, beta, e, 0, None)


def policy(lp=P, old=P, ref=None, adv=P, loss=P, weight=P, ws=P, n=BIG, B=20, S=9, lo=0.2, hi=0.2, c=0.0):
    return (lp, 9, old, 9, ref, 0, adv, 1, 0, None, 0, loss, P, P, weight, ws, n, B, S, lo, hi, c, 0, None)


@pytest.mark.parametrize("make,fn", [(tokens, "nq_token_logprobs"), (tokens_bwd, "nq_token_logprobs_bwd")])
def test_token_logprobs_refuses(make, fn):
    for kw in (dict(B=0), dict(S=0), dict(V=0), dict(V=-3)):
        refused(fn, INV, "sizes", *make(**kw))
    refused(fn, UNS, "dtype", *make(dt=7))
    refused(fn, INV, "strides", *make(rs=-1))
    refused(fn, INV, "required", *make(x=None))
    refused(fn, INV, "required", *make(labels=None))
    refused(fn, INV, "aligned", *make(x=ODD))
    refused(fn, UNS, "too many rows", *make(B=1 << 20, S=1 << 20))
    for t in (0.0, -1.0, float("inf"), float("nan"), 1e-45):
        refused(fn, INV, "temperature", *make(T=t))
    if fn.endswith("_bwd"):
        refused(fn, INV, "dlogits", *make(dx=None))
        refused(fn, INV, "dlogits", *make(dy=None))
        refused(fn, UNS, "too many rows", *make(B=1, S=(1 << 31) - 1, V=1 << 20))
    else:
        refused(fn, INV, "logprobs", *make(out=None))
        refused(fn, WS, "workspace", *make(V=20000, n=8))
        refused(fn, WS, "workspace", *make(V=20000, ws=None))


@pytest.mark.parametrize("make,fn", [(head, "nq_linear_logprobs"), (head_bwd, "nq_linear_logprobs_bwd")])
def test_linear_logprobs_refuses(make, fn):
    for kw in (dict(B=0), dict(S=0), dict(V=0), dict(H=0)):
        refused(fn, INV, "sizes", *make(**kw))
    refused(fn, UNS, "multiple of 8", *make(H=60))
    for kw in (dict(S=(1 << 24) + 1), dict(B=1 << 13, S=1 << 12), dict(V=(1 << 24) + 1), dict(H=(1 << 20) + 8)):
        refused(fn, UNS, "2^24", *make(**kw))
    for kw in (dict(x=None), dict(w=None), dict(labels=None), dict(stats=None)):
        refused(fn, INV, "required", *make(**kw))
    for kw in (dict(x=ctypes.c_void_p((1 << 20) + 8)), dict(w=ctypes.c_void_p((1 << 20) + 8)), dict(rs=60), dict(bs=4), dict(rs=-64)):
        refused(fn, INV, "aligned", *make(**kw))
    for t in (0.0, float("inf"), 1e-45):
        refused(fn, INV, "temperature", *make(T=t))
    for kw in (dict(ws=None), dict(n=100), dict(ws=ctypes.c_void_p((1 << 20) + 16))):
        refused(fn, WS, "workspace", *make(**kw))
    # kept: too small, misaligned, or for sizes that keep nothing
    wide = dict(H=256, rs=256)
    refused(fn, WS, "kept", *make(S=100, kept=P, nk=16, **wide))
    refused(fn, WS, "kept", *make(S=100, kept=ctypes.c_void_p((1 << 20) + 16), nk=BIG, **wide))
    refused(fn, WS, "kept", *make(S=64, kept=P, nk=BIG, **wide))
    refused(fn, WS, "kept", *make(S=100, kept=P, nk=BIG))
    if fn.endswith("_bwd"):
        refused(fn, INV, "dlogprobs", *make(dy=None))
        refused(fn, INV, "aligned", *make(dw=ctypes.c_void_p((1 << 20) + 8)))
        # nothing asked for: nothing done
        assert _lib.load().nq_linear_logprobs_bwd(*make(dh=None, dw=None)) == _lib.NQ_OK
    else:
        refused(fn, INV, "logprobs", *make(out=None))


def test_preference_loss_refuses():
    fn = "nq_preference_loss"
    for kw in (dict(B=0), dict(Sc=-1), dict(Sr=-1)):
        refused(fn, INV, "lengths", *preference(**kw))
    refused(fn, UNS, "too many tokens", *preference(Sc=1 << 40))
    refused(fn, UNS, "kind", *preference(kind=3))
    for b in (0.0, -1.0, float("inf"), float("nan")):
        refused(fn, INV, "beta", *preference(beta=b))
    for kw in (dict(e=-0.1), dict(e=0.5), dict(e=float("nan")), dict(e=0.1, kind=1), dict(e=0.1, kind=2)):
        refused(fn, INV, "label_smoothing", *preference(**kw))
    for kw in (dict(c=None), dict(r=None), dict(loss=None), dict(wc=None), dict(wr=None)):
        refused(fn, INV, "required", *preference(**kw))
    refused(fn, INV, "coef", *preference(coef=None))
    refused(fn, WS, "workspace", *preference(n=8))
    refused(fn, WS, "workspace", *preference(ws=None))
    refused("nq_preference_loss_bwd", INV, "dloss", P, None, None, 0, None, 0, P, P, 2, 3, 3, None)
    refused("nq_preference_loss_bwd", INV, "coef", None, P, None, 0, None, 0, P, P, 2, 3, 3, None)
    # no gradient asked for, or no tokens: nothing done
    for args in ((P, P, None, 0, None, 0, None, None, 2, 3, 3, None), (P, P, None, 0, None, 0, P, P, 2, 0, 0, None)):
        assert _lib.load().nq_preference_loss_bwd(*args) == _lib.NQ_OK


def test_policy_loss_refuses():
    fn = "nq_policy_loss"
    for kw in (dict(B=0), dict(S=-1)):
        refused(fn, INV, "must be positive", *policy(**kw))
    refused(fn, UNS, "too many tokens", *policy(S=1 << 40))
    for kw in (dict(lp=None), dict(old=None), dict(adv=None), dict(weight=None)):
        refused(fn, INV, "required", *policy(**kw))
    for kw in (dict(lo=-0.1), dict(lo=1.1), dict(hi=-0.1), dict(hi=float("inf")), dict(c=float("nan"))):
        refused(fn, INV, "clip_low", *policy(**kw))
    refused(fn, INV, "reference", *policy(c=0.1))
    refused(fn, INV, "loss", *policy(loss=None))
    refused(fn, WS, "workspace", *policy(n=8))
    refused(fn, WS, "workspace", *policy(ws=None))
    bwd = (P, 9, P, 9, None, 0, P, 1, 0, None, 0, P, None, P, 2, 9, 0.2, 0.2, 0.0, None)
    refused("nq_policy_loss_bwd", INV, "dloss", *bwd)


def test_workspaces():
    lib = _lib.load()
    assert lib.nq_token_logprobs_workspace_bytes(0, 10) == 0 and lib.nq_token_logprobs_workspace_bytes(5000, 151936) == 0
    assert lib.nq_token_logprobs_workspace_bytes(1, 151936) == 38 * 8   # slices of at least 4096 entries
    for rows in (0, 1 << 25):
        assert lib.nq_linear_logprobs_workspace_bytes(rows, 100, 64) == 0
        assert lib.nq_linear_logprobs_bwd_workspace_bytes(rows, 100, 64) == 0
    # kept: two bytes an entry, four a row and a maximum per 128 entries, each part from a multiple of 256
    def up(n):
        return -(-n // 256) * 256
    assert lib.nq_linear_logprobs_kept_bytes(65, 1001, 256) == up(65 * 4) + up(65 * 8 * 4) + up(65 * 1008 * 2)
    assert lib.nq_linear_logprobs_kept_bytes(64, 1001, 256) == 0
    assert lib.nq_linear_logprobs_kept_bytes(65, 1001, 248) == 0
    assert lib.nq_linear_logprobs_kept_bytes(16384, 151936, 256) == 0    # over 4 GiB
    # the backward's gradient of the logits is held at most 1 GiB at a time, however many rows
    small, large = (lib.nq_linear_logprobs_bwd_workspace_bytes(r, 151936, 64) for r in (2048, 1 << 16))
    assert small < 2 ** 31 and large < 2 ** 31 + 2 ** 28


def test_host_tensors_raise():
    x, y = torch.zeros(2, 8), torch.zeros(2, dtype=torch.long)
    for call in (lambda: nq.token_logprobs(x, y), lambda: nq.linear_logprobs(x.bfloat16(), x.bfloat16(), y),
                 lambda: nq.preference_loss(x, x), lambda: nq.policy_loss(x, x, x[:, 0])):
        with pytest.raises(RuntimeError, match="HIP device"):
            call()


# ---------------------------------------------------------------- calls with the kernels stubbed

@pytest.fixture
def stubbed(monkeypatch):
    """The operators on host tensors, with a library that counts its launches and writes nothing."""
    launches = []

    class Library:
        def __getattr__(self, name):
            if name.endswith("_bytes"):
                return lambda *args: 16
            return lambda *args: launches.append(name) or 0

    monkeypatch.setattr(_lib, "load", lambda: Library())
    monkeypatch.setattr(nq.losses.ops, "_require_device", lambda *ts: None)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: -1)
    return launches


def loss_calls():
    """Each operator as a function of its first operand, and one."""
    y, lp = torch.tensor([1, 2, 0]), torch.zeros(3, 4)
    w = torch.zeros(5, 8, dtype=torch.bfloat16)
    return {
        "token_logprobs": (lambda x: nq.token_logprobs(x, y), torch.zeros(3, 4)),
        "linear_logprobs": (lambda h: nq.linear_logprobs(h, w, y), torch.zeros(3, 8, dtype=torch.bfloat16)),
        "preference_loss": (lambda x: nq.preference_loss(x, lp, lp, lp)[0], torch.zeros(3, 4)),
        "policy_loss": (lambda x: nq.policy_loss(x, lp, lp[:, 0])[0], torch.zeros(3, 4)),
    }


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning", "ignore:.*jit.*:DeprecationWarning")
@pytest.mark.parametrize("name", ["token_logprobs", "linear_logprobs", "preference_loss", "policy_loss"])
def test_traces_are_refused(stubbed, name):
    """A trace would hold the allocation of the outputs without the kernel that writes them."""
    from torch.fx.experimental.proxy_tensor import make_fx
    call, x = loss_calls()[name]
    call(x)
    assert len(stubbed) == 1
    with pytest.raises(RuntimeError, match="trace"):
        torch.jit.trace(call, (x,), check_trace=False)
    for kw in ({}, dict(pre_dispatch=True)):
        with pytest.raises(RuntimeError, match="trace"):
            make_fx(call, **kw)(x)
    # a traced backward of an eager forward
    leaf = x.clone().requires_grad_()
    out = call(leaf)
    with pytest.raises(RuntimeError, match="trace"):
        make_fx(lambda d: torch.autograd.grad(out, leaf, d, retain_graph=True))(torch.ones_like(out))
    assert len(stubbed) == 2
    torch.autograd.grad(out, leaf, torch.ones_like(out))
    assert len(stubbed) == 3


def test_tensors_without_memory_are_refused(stubbed):
    """A wrapped tensor's null pointer stands for an operand left out: no mask, no reference."""
    from torch.testing._internal.two_tensor import TwoTensor
    for call, x in loss_calls().values():
        with pytest.raises((TypeError, RuntimeError)):
            torch.func.functionalize(call)(x)
        with pytest.raises(TypeError, match="memory"):
            call(TwoTensor(x, x))
    x = torch.zeros(3, 4)
    m = TwoTensor(x.bool(), x.bool())
    r = TwoTensor(x, x)
    for call in (lambda: nq.preference_loss(x, x, chosen_mask=m), lambda: nq.preference_loss(x, x, r, r),
                 lambda: nq.policy_loss(x, x, x, mask=m), lambda: nq.policy_loss(x, x, x, ref_logprobs=r)):
        with pytest.raises(TypeError, match="memory"):
            call()
    assert not stubbed
    # no elements need no memory
    nq.preference_loss(x[:, :0], x, chosen_mask=x[:, :0].bool())
    nq.policy_loss(x[:, :0], x[:, :0], x[:, 0])
    assert len(stubbed) == 2


@pytest.mark.parametrize("over", [2 ** 31, 2 ** 32 + 4])
def test_sizes_past_an_int_are_refused(stubbed, over):
    """ctypes would cut them to 32 bits: 2^32 + 4 sequences to the first 4, a width of 2^32 + 8 to 8."""
    many = torch.zeros(1).expand(over)
    with pytest.raises(ValueError, match="sequences"):
        nq.preference_loss(many, many)
    with pytest.raises(ValueError, match="sequences"):
        nq.policy_loss(many[:, None], many[:, None], many)
    one = torch.zeros(1, dtype=torch.bfloat16)
    for H in (over + 8 - over % 8, (1 << 20) + 8):
        with pytest.raises(ValueError, match="2.20"):
            nq.linear_logprobs(one.expand(3, H), one.expand(5, H), torch.zeros(3, dtype=torch.long))
    with pytest.raises(ValueError, match="2.24"):
        nq.linear_logprobs(one.expand(3, 8), one.expand(over, 8), torch.zeros(3, dtype=torch.long))
    with pytest.raises(ValueError, match="2.31"):
        nq.token_logprobs(torch.zeros(1).expand(3, over), torch.zeros(3, dtype=torch.long))
    assert not stubbed


def test_linear_logprobs_backward_refuses_more_hidden_states_than_a_launch_writes():
    """A thread writes 8 of the gradient's elements, and a launch of 2^32 threads would come out short."""
    fn = "nq_linear_logprobs_bwd"
    refused(fn, UNS, "hidden states", *head_bwd(S=1 << 24, H=2048, rs=2048))
    refused(fn, UNS, "hidden states", *head_bwd(S=(1 << 23) + 1, H=4096, rs=4096))
    refused(fn, UNS, "tiles", *head_bwd(S=1 << 24, H=1 << 20, rs=1 << 20))


def test_linear_logprobs_backward_workspace_of_many_rows():
    """The gradient of the logits: at most 1 GiB at a time up to 2^21 rows, 256 entries (512 bytes) a row beyond."""
    def ws(rows, V):
        return _lib.load().nq_linear_logprobs_bwd_workspace_bytes(rows, V, 64)
    for rows in (1, 4096, 1 << 16, (1 << 20) + 1, 1 << 21):
        assert ws(rows, 151936) - ws(rows, 8) <= 2 ** 30
    for rows in ((1 << 21) + 1, 1 << 22, 1 << 24):
        assert ws(rows, 151936) == ws(rows, 256)
        assert ws(rows, 256) - ws(rows, 8) <= 512 * rows


def test_negative_views_are_refused(stubbed):
    """The imaginary part of a conjugate holds the opposite of what it stands for."""
    lp = torch.complex(torch.zeros(3, 4), torch.ones(3, 4)).conj().imag
    assert lp.is_neg() and float(lp[0, 0]) == -1
    x, y, a = torch.zeros(3, 4), torch.tensor([1, 2, 0]), lp[:, 0]
    whole = torch._neg_view(x)
    for call in (lambda: nq.token_logprobs(whole, y), lambda: nq.preference_loss(whole, x), lambda: nq.preference_loss(a, a),
                 lambda: nq.preference_loss(x, x, x, whole), lambda: nq.policy_loss(x, x, a),
                 lambda: nq.policy_loss(x, x, whole), lambda: nq.policy_loss(x, whole, x),
                 lambda: nq.linear_logprobs(torch.zeros(3, 8, dtype=torch.bfloat16),
                                            torch._neg_view(torch.zeros(5, 8, dtype=torch.bfloat16)), y)):
        with pytest.raises(TypeError, match="resolve_neg"):
            call()
    assert not stubbed
    nq.policy_loss(x, lp.resolve_neg(), a.resolve_neg())
    nq.policy_loss(x, lp, x)  # whose rows are no vectors: copied, and resolved so
    assert len(stubbed) == 2 and not lp.contiguous().is_neg() and float(lp.contiguous()[0, 0]) == -1


def test_more_sequences_than_an_int_steps_over_are_refused(monkeypatch):
    """The threads that finish a loss step over its sequences by 256 in an int, which would pass its end."""
    for B in ((1 << 30) + 1, (1 << 31) - 1):
        refused("nq_preference_loss", UNS, "sequences", *preference(B=B))
        refused("nq_policy_loss", UNS, "sequences", *policy(B=B))
        refused("nq_preference_loss_bwd", UNS, "sequences", P, P, None, 0, None, 0, P, P, B, 1, 1, None)
        refused("nq_policy_loss_bwd", UNS, "sequences", P, 9, P, 9, None, 0, P, 1, 0, None, 0, P, P, P, B, 1, 0.2,
                   0.2, 0.0, None)
    monkeypatch.setattr(nq.losses.ops, "_require_device", lambda *ts: None)
    many = torch.zeros(1).expand((1 << 30) + 1)
    with pytest.raises(ValueError, match="sequences"):
        nq.preference_loss(many, many)
    with pytest.raises(ValueError, match="sequences"):
        nq.policy_loss(many[:, None], many[:, None], many)
