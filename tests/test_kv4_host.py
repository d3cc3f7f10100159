"""The 4-bit cache and eviction without a GPU: refusals, bookkeeping, the work's division."""

import ctypes
import random

import pytest
import torch

import nano_qwen_amd as nq
from nano_qwen_amd import _lib, attention, kv4
from tests import kv4_reference as ref

A = ctypes.c_void_p(1 << 20)            # aligned addresses, never followed: every call here is refused
A2 = ctypes.c_void_p(1 << 21)
ODD = ctypes.c_void_p((1 << 20) + 4)


def i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


S3 = i64(4096, 1024, 128)
POOL = i64(64 * 136 * 4, 64 * 136)      # pages of 4 heads, 64 rows of 128 in 136 bytes each
BF16, F32 = _lib.NQ_DTYPE_BF16, _lib.NQ_DTYPE_F32

APPEND = dict(k=A, ks=S3, v=A, vs=S3, q=None, qs=None, qo=None, qos=None, pool=A, ps=POOL, pages=8, bt=A, bts=4, cols=4,
              page=64, B=2, S=3, Hq=0, Hkv=4, D=128, dtype=BF16, qw=None, kw=None, eps=1e-6, cos=None, sin=None, max_pos=0,
              pos=None, pos_base=None, pos_shift=None, pos0=0, row_base=A, row0=0, lens_out=None, stream=None)
GATHER = dict(pool=A, ps=POOL, pages=8, bt=A, bts=4, cols=4, page=64, k=A, ks=S3, v=A, vs=S3, B=2, S=3, Hkv=4, D=128,
              dtype=BF16, row_base=None, row0=0, stream=None)
DECODE = dict(q=A, qs=i64(1024, 128), pool=A, ps=POOL, pages=8, bt=A, bts=4, cols=4, page=64, lens=A, o=A,
              os=i64(1024, 128), lse=None, ws=A, wsb=1 << 30, B=2, Hq=8, Hkv=4, D=128, max_len=200, dtype=BF16, scale=0.0,
              stream=None)
SHARED = dict(DECODE, cols=1000, bts=1000, max_len=64000)
WEIGHTS = dict(q=A, qs=S3, pool=A, ps=i64(32768, 8192, 128), four=0, pages=8, bt=A, bts=4, cols=4, page=64, lens=A, lse=A,
               w=A, ws=i64(1024, 256), add=0, work=A, workb=1 << 30, B=2, Hq=8, Hkv=4, S=300, D=128, max_len=200, causal=1,
               scale=0.0, stream=None)
SELECT = dict(w=A, ws=i64(1024, 256), lens=A, kept=A, B=2, H=4, W=256, keep=100, recent=10, first=4, stream=None)
COMPACT = dict(k=A, ks=POOL, v=None, vs=None, row=0, D=128, pages=8, bt=A, bts=4, cols=4, new=A2, nbts=2, ncols=2, page=64,
               kept=A, w=None, wo=None, ws=None, W=0, B=2, H=4, keep=100, stream=None)
PLAIN = dict(COMPACT, ks=i64(65536, 16384, 256), v=A, vs=i64(65536, 16384, 256), row=256)

REFUSED = [
    ("nq_kv4_append", APPEND, dict(D=96), b"head_dim"),
    ("nq_kv4_append", APPEND, dict(D=0), b"head_dim"),
    ("nq_kv4_append", APPEND, dict(page=48), b"page_size"),
    ("nq_kv4_append", APPEND, dict(page=0), b"page_size"),
    ("nq_kv4_append", APPEND, dict(page=1 << 21), b"page_size"),
    ("nq_kv4_append", APPEND, dict(pool=None), b"required"),
    ("nq_kv4_append", APPEND, dict(bt=None), b"required"),
    ("nq_kv4_append", APPEND, dict(pool=ODD), b"16 bytes"),
    ("nq_kv4_append", APPEND, dict(ps=i64(64 * 136 * 4, 64 * 135)), b"overlap"),
    ("nq_kv4_append", APPEND, dict(pages=0), b"num_pages"),
    ("nq_kv4_append", APPEND, dict(bts=3), b"bt_cols"),
    ("nq_kv4_append", APPEND, dict(B=0), b"positive"),
    ("nq_kv4_append", APPEND, dict(S=-1), b"positive"),
    ("nq_kv4_append", APPEND, dict(dtype=7), b"dtype"),
    ("nq_kv4_append", APPEND, dict(k=ODD), b"aligned"),
    ("nq_kv4_append", APPEND, dict(ks=i64(4096, 1024, 127)), b"strides"),
    ("nq_kv4_append", APPEND, dict(cos=A), b"together"),
    ("nq_kv4_append", APPEND, dict(cos=A, sin=ODD, max_pos=4), b"aligned"),
    ("nq_kv4_append", APPEND, dict(kw=ODD), b"aligned"),
    ("nq_kv4_append", APPEND, dict(lens_out=A), b"alias"),
    ("nq_kv4_append", APPEND, dict(lens_out=A2, pos_base=A2), b"alias"),
    ("nq_kv4_append", APPEND, dict(lens_out=A2, pos_shift=A2), b"alias"),
    ("nq_kv4_append", APPEND, dict(B=1 << 15, S=1 << 12), b"too many rows"),
    ("nq_kv4_gather", GATHER, dict(v=None), b"required"),
    ("nq_kv4_gather", GATHER, dict(dtype=2), b"dtype"),
    ("nq_kv4_gather", GATHER, dict(vs=i64(1, 1, 1)), b"strides"),
    ("nq_kv4_gather", GATHER, dict(B=1 << 10, S=1 << 20), b"too many rows"),
    ("nq_kv4_gather", GATHER, dict(S=0), b"positive"),
    ("nq_attn_decode_kv4", DECODE, dict(Hq=9), b"divisible"),
    ("nq_attn_decode_kv4", DECODE, dict(Hq=0), b"positive"),
    ("nq_attn_decode_kv4", DECODE, dict(max_len=257), b"columns"),
    ("nq_attn_decode_kv4", DECODE, dict(max_len=0), b"positive"),
    ("nq_attn_decode_kv4", DECODE, dict(lens=None), b"required"),
    ("nq_attn_decode_kv4", DECODE, dict(q=ODD), b"aligned"),
    ("nq_attn_decode_kv4", DECODE, dict(os=i64(1024, 4)), b"strides"),
    ("nq_attn_decode_kv4", SHARED, dict(wsb=1000), b"workspace"),
    ("nq_attn_decode_kv4", SHARED, dict(ws=None), b"workspace"),
    ("nq_attn_decode_kv4", SHARED, dict(ws=ODD), b"workspace"),
    ("nq_attn_decode_kv4", DECODE, dict(dtype=3), b"dtype"),
    ("nq_attn_decode_kv4", DECODE, dict(B=1 << 20), b"one launch"),
    ("nq_key_weights", WEIGHTS, dict(D=48), b"head_dim"),
    ("nq_key_weights", WEIGHTS, dict(Hq=7), b"divisible"),
    ("nq_key_weights", WEIGHTS, dict(max_len=300), b"columns"),
    ("nq_key_weights", WEIGHTS, dict(workb=16), b"workspace"),
    ("nq_key_weights", WEIGHTS, dict(lse=None), b"required"),
    ("nq_key_weights", WEIGHTS, dict(qs=i64(4096, 1024, -128)), b"strides"),
    ("nq_key_weights", WEIGHTS, dict(S=1 << 24), b"rows"),
    ("nq_key_weights", WEIGHTS, dict(page=100), b"page_size"),
    ("nq_select_keys", SELECT, dict(keep=0), b"keep"),
    ("nq_select_keys", SELECT, dict(recent=97), b"keep"),
    ("nq_select_keys", SELECT, dict(first=-1), b"keep"),
    ("nq_select_keys", SELECT, dict(w=None), b"required"),
    ("nq_select_keys", SELECT, dict(B=0), b"positive"),
    ("nq_select_keys", SELECT, dict(B=1 << 20), b"one launch"),
    ("nq_kv_compact", COMPACT, dict(new=A), b"new"),
    ("nq_kv_compact", COMPACT, dict(ncols=1, nbts=1), b"kept"),
    ("nq_kv_compact", COMPACT, dict(D=256), b"head_dim"),
    ("nq_kv_compact", COMPACT, dict(w=A), b"together"),
    ("nq_kv_compact", COMPACT, dict(w=A, wo=A, ws=i64(512, 128), W=128), b"weights_out"),
    ("nq_kv_compact", COMPACT, dict(w=A, wo=A2, ws=i64(512, 128), W=64), b"together"),
    ("nq_kv_compact", COMPACT, dict(keep=0), b"positive"),
    ("nq_kv_compact", COMPACT, dict(keep=1 << 30, ncols=1 << 25, nbts=1 << 25), b"one launch"),
    ("nq_kv_compact", PLAIN, dict(row=100), b"16 bytes"),
    ("nq_kv_compact", PLAIN, dict(ks=i64(65536, 16384, 128)), b"overlap"),
    ("nq_kv_compact", PLAIN, dict(v=ODD), b"16 bytes"),
]


@pytest.mark.parametrize("fn,base,change,text", REFUSED)
def test_c_entries_refuse(fn, base, change, text):
    lib = _lib.load()
    assert set(change) <= set(base) and len(base) == len(_lib.SIGNATURES[fn][1])
    rc = getattr(lib, fn)(*dict(base, **change).values())
    assert rc != _lib.NQ_OK and text in lib.nq_last_error(), lib.nq_last_error()


def test_workspaces():
    lib = _lib.load()
    rows = 64 * 4
    assert lib.nq_attn_decode_kv4_workspace_bytes(64, 64, 4, 128, 32768) == (512 + rows) * 16 * 130 * 4 + rows * 8
    assert lib.nq_attn_decode_kv4_workspace_bytes(64, 65, 4, 128, 32768) == 0
    assert lib.nq_attn_decode_kv4_workspace_bytes(1, 16, 8, 128, 512) == 0   # whole rows a workgroup
    assert lib.nq_key_weights_workspace_bytes(2, 8, 4, 1, 200) == 0      # 2 rows: no partial sums
    assert lib.nq_key_weights_workspace_bytes(2, 8, 4, 128, 200) == 0    # one chunk
    assert lib.nq_key_weights_workspace_bytes(2, 8, 4, 129, 200) == 2 * 2 * 4 * 200 * 4


@pytest.fixture
def host_calls(monkeypatch):
    """The Python checks on host tensors; a call that passes them would raise."""
    def reached(plan, t, fn, args, name, keep, result):
        raise AssertionError(f"{name} was not refused")
    monkeypatch.setattr(kv4, "_check", lambda *a: None)
    monkeypatch.setattr(kv4, "_launch", reached)


def pool4(n=4, H=2, P=32, D=64):
    return kv4.kv4_empty_pool(n, H, P, D, device="cpu")


def rows(B=1, H=2, S=3, D=64, dtype=torch.bfloat16):
    return torch.zeros(B, H, S, D, dtype=dtype)


TABLE = torch.zeros(1, 3, dtype=torch.int32)
LENS = torch.ones(1, dtype=torch.int32)


@pytest.mark.parametrize("change,error", [
    (dict(k=rows(H=3), v=rows(H=3)), ValueError), (dict(v=rows(S=2)), ValueError), (dict(v=rows(dtype=torch.float32)), TypeError),
    (dict(k=rows(D=32), v=rows(D=32)), ValueError), (dict(k=rows(dtype=torch.float16), v=rows(dtype=torch.float16)), TypeError),
    (dict(pool=torch.zeros(4, 2, 32, 64)), ValueError), (dict(pool=torch.zeros(4, 2, 32, 67, dtype=torch.uint8)), ValueError),
    (dict(pool=torch.zeros(4, 2, 40, 68, dtype=torch.uint8)), ValueError), (dict(pool=pool4()[..., :34]), ValueError),
    (dict(pool=pool4().transpose(1, 2)), ValueError), (dict(block_table=TABLE.expand(2, 3)), ValueError),
    (dict(block_table=TABLE[0]), ValueError), (dict(row_offset=94), ValueError), (dict(row_offset=-1), ValueError),
    (dict(q=rows(S=2)), ValueError), (dict(q=rows(dtype=torch.float32)), TypeError), (dict(q_out=rows()), ValueError),
    (dict(q=rows(), q_out=rows(H=4)), ValueError), (dict(q=rows(), q_out=rows().transpose(2, 3).contiguous().transpose(2, 3)), ValueError),
    (dict(q_weight=torch.ones(64)), ValueError), (dict(k_weight=torch.ones(63)), ValueError), (dict(cos=torch.ones(8, 32)), ValueError),
    (dict(cos=torch.ones(8, 16), sin=torch.ones(8, 16)), ValueError), (dict(cos=torch.ones(8, 32), sin=torch.ones(8, 32), pos_offset=6), IndexError),
    (dict(lens_out=LENS), ValueError), (dict(lens_out=LENS, row_base=LENS), ValueError),
    (dict(lens_out=LENS, row_base=LENS.clone(), pos_base=LENS), ValueError),
    (dict(lens_out=LENS, row_base=LENS.clone(), pos_shift=LENS), ValueError),
    (dict(lens_out=LENS.long(), row_base=LENS), ValueError), (dict(row_base=LENS.expand(2)), ValueError),
    (dict(pos_shift=LENS.expand(3)), ValueError),
])
def test_append_refuses(host_calls, change, error):
    args = dict(k=rows(), v=rows(), pool=pool4(), block_table=TABLE)
    args.update(change)
    with pytest.raises(error):
        kv4.kv4_append(args.pop("k"), args.pop("v"), args.pop("pool"), args.pop("block_table"), **args)


@pytest.mark.parametrize("change,error", [
    (dict(S=97), ValueError), (dict(S=-1), ValueError), (dict(S=3, row_offset=94), ValueError), (dict(S=3, dtype=torch.float16), TypeError),
    (dict(S=3, k_out=rows(S=4)), ValueError), (dict(S=3, v_out=rows(dtype=torch.float32)), ValueError),
    (dict(S=3, row_base=torch.zeros(2, dtype=torch.int32)), ValueError),
])
def test_gather_refuses(host_calls, change, error):
    with pytest.raises(error):
        kv4.kv4_gather(pool4(), TABLE, **change)


@pytest.mark.parametrize("change,error", [
    (dict(q=torch.zeros(1, 3, 64, dtype=torch.bfloat16)), ValueError), (dict(q=rows(S=2)), ValueError), (dict(q=rows(D=32)[:, :, 0]), ValueError),
    (dict(q=torch.zeros(1, 2, 64, dtype=torch.float16)), TypeError), (dict(max_len=0), ValueError), (dict(max_len=97), ValueError),
    (dict(lens=LENS.expand(2)), ValueError), (dict(out=torch.zeros(1, 2, 64)), ValueError), (dict(q=torch.zeros(1, 0, 64)), ValueError),
    (dict(workspace=torch.zeros(1, dtype=torch.uint8).expand(1 << 24)), ValueError),
])
def test_decode_refuses(host_calls, change, error):
    args = dict(q=torch.zeros(1, 2, 64, dtype=torch.bfloat16), pool=pool4(), block_table=TABLE, lens=LENS, max_len=90)
    args.update(change)
    with pytest.raises(error):
        kv4.attention_decode_kv4(args.pop("q"), args.pop("pool"), args.pop("block_table"), args.pop("lens"), **args)


@pytest.mark.parametrize("change,error", [
    (dict(q=rows(dtype=torch.float32)), TypeError), (dict(q=rows(H=3)), ValueError), (dict(k_pool=torch.zeros(4, 2, 32, 64)), TypeError),
    (dict(k_pool=torch.zeros(4, 2, 40, 64, dtype=torch.bfloat16)), ValueError), (dict(lse=torch.zeros(1, 2, 2)), ValueError),
    (dict(lse=torch.zeros(1, 2, 3, dtype=torch.float64)), ValueError), (dict(max_len=97), ValueError),
    (dict(weights=torch.zeros(1, 2, 89)), ValueError), (dict(weights=torch.zeros(1, 2, 90, dtype=torch.float64)), ValueError),
    (dict(weights=torch.zeros(1, 90, 2).transpose(1, 2)), ValueError), (dict(lens=LENS.expand(2)), ValueError),
    (dict(weights=torch.zeros(1, 1, 90).expand(1, 2, 90)), ValueError), (dict(weights=torch.zeros(200).as_strided((1, 2, 90), (0, 89, 1))), ValueError),
])
def test_key_weights_refuse(host_calls, change, error):
    args = dict(q=rows(), k_pool=pool4(), block_table=TABLE, lens=LENS, lse=torch.zeros(1, 2, 3), max_len=90)
    args.update(change)
    with pytest.raises(error):
        first = [args.pop(n) for n in ("q", "k_pool", "block_table", "lens", "lse")]
        kv4.attention_key_weights(*first, **args)


@pytest.mark.parametrize("change,error", [
    (dict(keep=0), ValueError), (dict(keep=4, recent=3, first=2), ValueError), (dict(keep=4, recent=-1), ValueError),
    (dict(keep=2 ** 31), ValueError), (dict(weights=torch.zeros(2, 8)), ValueError), (dict(weights=torch.zeros(1, 2, 8).double()), ValueError),
    (dict(lens=LENS.expand(2)), ValueError),
])
def test_select_refuses(host_calls, change, error):
    args = dict(dict(weights=torch.zeros(1, 2, 8), lens=LENS, keep=4), **change)
    with pytest.raises(error):
        kv4.select_keys(args.pop("weights"), args.pop("lens"), **args)


@pytest.mark.parametrize("change,error", [
    (dict(kept=torch.zeros(1, 3, 4, dtype=torch.int32)), ValueError), (dict(kept=torch.zeros(1, 2, 4)), ValueError),
    (dict(kept=torch.zeros(1, 2, 33, dtype=torch.int32)), ValueError), (dict(new_table=TABLE[:, :1]), ValueError),
    (dict(weights=torch.zeros(1, 2, 3)), ValueError), (dict(pools=(torch.zeros(4, 2, 32, 64), torch.zeros(4, 2, 32, 32))), ValueError),
    (dict(pools=(torch.zeros(4, 2, 32, 64), torch.zeros(4, 2, 32, 64).bfloat16())), ValueError),
    (dict(pools=(torch.zeros(4, 2, 32, 64).half(),) * 2), TypeError), (dict(pools=(torch.zeros(4, 2, 40, 64),) * 2), ValueError),
])
def test_compact_refuses(host_calls, change, error):
    args = dict(pools=pool4(), block_table=TABLE, new_table=torch.ones(1, 1, dtype=torch.int32), kept=torch.zeros(1, 2, 4, dtype=torch.int32))
    args.update(change)
    with pytest.raises(error):
        first = [args.pop(n) for n in ("pools", "block_table", "new_table", "kept")]
        kv4.kv_compact(*first, **args)


def test_host_tensors_have_no_path():
    with pytest.raises(RuntimeError, match="no CPU path"):
        kv4.kv4_append(rows(), rows(), pool4(), TABLE)
    with pytest.raises(RuntimeError, match="no CPU path"):
        kv4.select_keys(torch.zeros(1, 2, 8), LENS, keep=4)
    for bad in (48, 16, 256, 33):
        with pytest.raises(ValueError, match="head_dim"):
            kv4.kv4_empty_pool(1, 1, 32, bad, device="cpu")
    with pytest.raises(ValueError, match="page_size"):
        kv4.kv4_empty_pool(1, 1, 48, 64, device="cpu")


def test_recordings_and_gradients_are_refused(monkeypatch):
    """A trace would hold the outputs' allocation without the launch; forward mode has no tangents."""
    monkeypatch.setattr(kv4.ops, "_require_device", lambda *a: None)
    lib = type("L", (), {n: staticmethod(lambda *a: 0) for n in _lib.SIGNATURES})
    monkeypatch.setattr(_lib, "load", lambda: lib)
    weights = torch.rand(1, 2, 8)
    with pytest.raises(RuntimeError, match="trace"):
        torch.jit.trace(lambda w: kv4.select_keys(w, LENS, keep=4), (weights,), check_trace=False)
    from torch.fx.experimental.proxy_tensor import make_fx
    with pytest.raises(RuntimeError):
        make_fx(lambda w: kv4.select_keys(w, LENS, keep=4))(weights)
    with pytest.raises(RuntimeError, match="no gradient"):
        kv4.select_keys(weights.clone().requires_grad_(), LENS, keep=4)
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        kv4.select_keys(fwd.make_dual(weights, weights), LENS, keep=4)


@pytest.mark.parametrize("current", [0, 3])
def test_launches_go_to_the_tensors_device_and_its_stream(monkeypatch, current):
    seen = []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            seen.append(("enter", self.index))

        def __exit__(self, *a):
            seen.append(("exit", self.index))
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 1000 + i, raising=False)
    monkeypatch.setattr(torch.cuda, "device", Device)
    t = type("T", (), dict(get_device=lambda self: 3, device=torch.device("cuda", 3)))()
    fn = lambda *a: seen.append(a) or 0  # noqa: E731
    around = lambda call: [("enter", 3), call, ("exit", 3)] if current != 3 else [call]  # noqa: E731
    assert kv4._launch(False, t, fn, (1, 2), "f", (), "result") == "result"
    assert seen == around((1, 2, 1003))
    seen.clear()
    plan = kv4._launch(True, t, fn, (1, 2), "f", (), "result")
    assert seen == [] and plan.launch() == "result" and seen == around((1, 2, 1003))


# ---------------------------------------------------------------- the caches' bookkeeping
@pytest.fixture
def plain_eviction(monkeypatch):
    """select_keys and kv_compact by their definitions, on host tensors."""
    def select_keys(weights, lens, *, keep, recent, first):
        out = torch.full((*weights.shape[:2], keep), -1, dtype=torch.int32)
        for b in range(out.shape[0]):
            for h in range(out.shape[1]):
                got = ref.select(weights[b, h], int(lens[b]), keep, recent, first)
                out[b, h, :len(got)] = torch.tensor(got, dtype=torch.int32)
        return out

    def kv_compact(pools, table, new, kept, *, weights):
        out = torch.zeros_like(weights)
        P = pools[0].shape[2]
        old = [p.clone() for p in pools]
        for b in range(kept.shape[0]):
            rows = int(kept[b].max()) + 1
            assert not set(new[b].tolist()) & set(table[b, :-(-rows // P)].tolist())
            for h in range(kept.shape[1]):
                for i, j in enumerate(kept[b, h].tolist()):
                    for p, o in zip(pools, old):
                        p[new[b, i // P], h, i % P] = o[table[b, j // P], h, j % P]
                    out[b, h, i] = weights[b, h, j]
        return out
    monkeypatch.setattr(attention.kv4, "select_keys", select_keys)
    monkeypatch.setattr(attention.kv4, "kv_compact", kv_compact)


def filled(lens, num_pages=20, P=32, H=2, D=8, track=4):
    c = nq.PagedKVCache(num_pages, page_size=P, track_weights=track)
    c._setup(len(lens), H, D, torch.bfloat16, "cpu")
    c._grow(lens)
    c.host_lens = list(lens)
    c.lens.copy_(torch.tensor(lens, dtype=torch.int32))
    g = torch.Generator().manual_seed(1)
    for p in (c.k_pool, c.v_pool):
        p.copy_(torch.randn(p.shape, generator=g))
    for b, n in enumerate(lens):
        c.weights[b, :, :n] = torch.rand(H, n, generator=g)
    return c


def all_pages(c):
    return sorted(c._free + sum(c._pages, []))


@pytest.mark.parametrize("spare", [20, 3])
def test_evict_in_as_many_goes_as_pages_allow(plain_eviction, spare):
    lens = [90, 33, 70, 200]
    used = sum(-(-n // 32) for n in lens)
    c = filled(lens, num_pages=used + spare)
    held = [c.gather(b) for b in range(4)]
    w = c.weights.clone()
    calls = []
    real = c._evict_some
    c._evict_some = lambda rows, *a: (calls.append(list(rows)), real(rows, *a))
    c.evict(40, recent=8, first=3)
    assert calls == ([[0, 2, 3]] if spare == 20 else [[0], [2, 3]])
    assert c.host_lens == [40, 33, 40, 40] == c.lens.tolist() and c.evicted == [50, 0, 30, 160]
    assert c._shift.tolist() == c.evicted and c._next_positions().tolist() == [90, 33, 70, 200]
    assert all_pages(c) == list(range(used + spare)) and [len(p) for p in c._pages] == [2] * 4
    for b, n in enumerate(lens):
        k, v = c.gather(b)
        for h in range(2):
            keep = ref.select(w[b, h], n, 40, 8, 3) if n > 40 else list(range(n))
            assert torch.equal(k[h], held[b][0][h, keep]) and torch.equal(v[h], held[b][1][h, keep])
            assert torch.equal(c.weights[b, h, :len(keep)], w[b, h, keep]) and not c.weights[b, h, len(keep):].any()
    c.evict(40)  # nothing longer: nothing moves
    assert c.evicted == [50, 0, 30, 160] and len(calls) == (1 if spare == 20 else 2)


def test_evict_refuses(plain_eviction):
    c = filled([90, 33], num_pages=6)
    for bad in (dict(keep=0), dict(keep=4, recent=3, first=2), dict(keep=4, recent=-1), dict(keep=4, first=-1)):
        with pytest.raises(ValueError):
            c.evict(**bad)
    with pytest.raises(RuntimeError, match="out of pages"):
        c.evict(64)  # needs two free pages, one is
    assert c.host_lens == [90, 33] and c.free_pages == 1 and all_pages(c) == list(range(6))
    with pytest.raises(ValueError, match="track_weights"):
        nq.PagedKVCache(4, page_size=32).evict(1)
    with pytest.raises(ValueError):
        nq.PagedKVCache(4, page_size=32, track_weights=-1)
    for cls in (nq.PagedKVCache, nq.PagedKVCache4):
        with pytest.raises(TypeError, match="bfloat16"):
            cls(4, page_size=32, track_weights=1)._setup(1, 2, 64, torch.float32, "cpu")


def test_trimmed_and_freed_sequences_lose_their_weights(plain_eviction):
    c = filled([90, 70])
    w = c.weights.clone()
    c.set_lengths([50, 70])
    assert not c.weights[0, :, 50:].any() and torch.equal(c.weights[0, :, :50], w[0, :, :50])
    assert torch.equal(c.weights[1], w[1])
    c.evict(40)
    assert c.evicted == [10, 30]
    c.free(0)
    assert c.evicted == [0, 30] and not c.weights[0].any() and c._shift.tolist() == [0, 30]
    c.free(1)
    assert c._shift is None and c._next_positions() is None


def test_expected_lengths():
    c = filled([0, 0])
    for bad in ([0, 3], [-1, 2]):
        with pytest.raises(ValueError):
            c.expect_lengths(bad)
    c.expect_lengths(torch.tensor([3, 5]))
    with pytest.raises(ValueError, match="do not fit"):
        c._take_expected(2, 4)
    assert c._take_expected(2, 4) is None  # asked for once
    c.expect_lengths([3, 5])
    with pytest.raises(ValueError, match="do not fit"):
        c._take_expected(3, 8)
    c.expect_lengths([3, 5])
    assert c._take_expected(2, 5) == [3, 5]


def test_a_4_bit_cache_of_other_rows_refuses():
    c = nq.PagedKVCache4(4, page_size=32)
    c._setup(2, 2, 64, torch.bfloat16, "cpu")
    assert c.pool.shape == (4, 2, 32, 68) and c.pool.dtype == torch.uint8
    for H, D, dtype in ((4, 64, torch.bfloat16), (2, 128, torch.bfloat16), (2, 64, torch.float32)):
        with pytest.raises(ValueError, match="pool holds"):
            c._setup(2, H, D, dtype, "cpu")
    with pytest.raises(ValueError):
        nq.PagedKVCache4(4, page_size=32)._setup(2, 2, 96, torch.bfloat16, "cpu")


@pytest.mark.parametrize("kw", [dict(kv_bits=8), dict(kv_bits=4), dict(keep=64), dict(page_size=32, keep=0),
                                dict(page_size=32, keep=8, recent=8), dict(page_size=32, keep=8, recent=-1),
                                dict(page_size=32, keep=8, first=9, recent=0)])
def test_generator_refuses(kw):
    with pytest.raises(ValueError):
        nq.generate_greedy_batch(None, [[1]], 4, **kw)


# ---------------------------------------------------------------- the work's division
STEP, COST = 32, 24


def decode_split(lens, rows_per_batch, groups, least):
    """[(workgroup, row, first step, steps)] of the shared 4-bit decode, key steps only."""
    nb = [-(-n // STEP) + COST if n > 0 else 0 for n in lens]
    N = sum(nb) * rows_per_batch
    used, out = max(min(groups, N // least), 1) if N else 0, []
    starts = []  # (global step, row, steps)
    at = 0
    for b, n in enumerate(nb):
        for j in range(rows_per_batch if n else 0):
            starts.append((at, b * rows_per_batch + j, n))
            at += n
    for w in range(used):
        q0, q1 = w * N // used, (w + 1) * N // used
        assert q1 > q0
        for s, r, n in starts:
            a, z = max(q0, s), min(q1, s + n)
            if a < z:  # steps [a - s, z - s) of the row, of which the first COST hold no keys
                out.append((w, r, max(a - s - COST, 0), max(z - s - COST, 0) - max(a - s - COST, 0)))
    return out, nb


def test_shared_decode_covers_every_key_step_once():
    rng = random.Random(5)
    for _ in range(60):
        B, rpb = rng.choice([1, 2, 5, 17]), rng.choice([1, 2, 8])
        lens = [rng.choice([0, 1, 31, 32, 33, rng.randrange(1, 4000)]) for _ in range(B)]
        groups = rng.choice([1, 7, 64, 512])
        least = rng.choice([8, 9, 40])  # 8, or more for long rows
        parts, nb = decode_split(lens, rpb, groups, least)
        slots = set()
        for r in range(B * rpb):
            mine = [(w, a, n) for w, row, a, n in parts if row == r]
            steps = -(-lens[r // rpb] // STEP)
            assert sorted(s for _, a, n in mine for s in range(a, a + n)) == list(range(steps))
            ws = [w for w, _, _ in mine]
            assert ws == list(range(ws[0], ws[-1] + 1)) if ws else steps == 0  # the merge's run has no gap
            for w in ws:
                assert w + r < 512 + B * rpb and (w + r not in slots or len(ws) == 1)
                if len(ws) > 1:
                    slots.add(w + r)


def chunk_ranges(S, G, max_len, causal, chunk, d, rows=256):
    R = S * G
    end = (chunk + 1) * rows if R // rows > chunk else R
    seen = max_len - S + (end - 1) // G + 1 if causal else max_len
    return (seen + d - 1) // d if seen > 0 else 0


@pytest.mark.parametrize("causal", [False, True])
def test_key_weight_ranges_reach_every_seen_key(causal):
    rng = random.Random(6)
    for _ in range(200):
        S, G = rng.choice([3, 17, 300, rng.randrange(3, 5000)]), rng.choice([1, 2, 7, 16])
        max_len, d = rng.randrange(1, 6000), 256 * rng.randrange(1, 9)
        R = S * G
        if R <= 16:
            continue
        n = -(-R // 256)
        counts = [chunk_ranges(S, G, max_len, causal, c, d) for c in range(n)]
        assert counts == sorted(counts) and counts[-1] * d >= max_len
        for c in range(n):
            last = min((c + 1) * 256, R) - 1
            seen = max_len - S + last // G + 1 if causal else max_len  # keys that the chunk's last row sees
            assert counts[c] * d >= seen
        # the sum's search: the first chunk that reaches key t, found by halving
        for t in (0, max_len - 1, rng.randrange(max_len)):
            lo, hi = 0, n
            while lo < hi:
                mid = (lo + hi) // 2
                if counts[mid] <= t // d:
                    lo = mid + 1
                else:
                    hi = mid
            assert lo == next(c for c in range(n) if counts[c] > t // d)


def test_multiplied_divisions_are_exact():
    """floor(n / d) by n * floor(2^32 / d) >> 32 and one correction, for n < 2^31."""
    rng = random.Random(7)
    for _ in range(20000):
        d = rng.choice([1, 2, 3, 255, 256, 2 ** 20, rng.randrange(1, 2 ** 31)])
        n = rng.choice([0, 1, 2 ** 31 - 1, rng.randrange(2 ** 31), min(2 ** 31 - 1, d * rng.randrange(1, 1 + 2 ** 31 // d)),
                        max(0, min(2 ** 31 - 1, d * rng.randrange(1, 1 + 2 ** 31 // d)) - 1)])
        m = 0xffffffff if d == 1 else 2 ** 32 // d
        q = n * m >> 32
        q += n - q * d >= d
        assert q == n // d


def test_quantiser_definition():
    """The scale is the smallest of which the block's largest is at most 7 times, and no element is
    off by more than a fifth of the largest: by (y - 4) / y or (6 - y) / y for y of 4 to 6 scales,
    1/7 for 7, half a scale of more than 3.5 below."""
    g = torch.Generator().manual_seed(8)
    x = torch.randn(500, 64, generator=g) * torch.exp2(torch.randint(-20, 20, (500, 1), generator=g).float())
    codes, byte = ref.quantise(x)
    amax = x.reshape(500, 2, 32).abs().amax(-1).double()
    scale = torch.exp2(byte.double() - 127)
    assert (amax <= 7 * scale).all() and (amax > 3.5 * scale).all()
    err = (ref.values(codes, byte) - x.double()).abs().reshape(500, 2, 32)
    assert (err <= scale[..., None]).all()
    assert (err <= amax[..., None] / 5).all()


# ---------------------------------------------------------------- operands that have to be copied
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_of_any_layout_are_read_in_place_or_copied_once(dtype):
    """Among them contiguous tensors that `contiguous()` would return as they are."""
    base = torch.arange(2 * 4 * 3 * 128 + 8, dtype=torch.float32).to(dtype)
    n = 2 * 4 * 3 * 128
    off = base[1:1 + n].view(2, 4, 3, 128)
    assert off.is_contiguous() and off.data_ptr() % 16
    odd_axis = base[:2 * 4 * 128].as_strided((2, 1, 4, 128), (512, 131, 128, 1))
    odd_outer = base[:4 * 3 * 128].as_strided((1, 4, 3, 128), (7, 384, 128, 1))
    swapped = base[:n].view(2, 4, 128, 3).transpose(2, 3)
    wide = base[:2 * 4 * 3 * 128].view(2, 4, 3, 128)[..., 1:65]
    for t in (off, odd_axis, odd_outer, swapped, wide):
        got, at, strides = kv4._rows(t)
        assert torch.equal(got, t) and at == got.data_ptr() and at % 16 == 0 and list(strides) == list(got.stride()[:-1])
        assert got.stride(-1) == 1 and all(s * got.element_size() % 16 == 0 for s in got.stride()[:-1])
        assert got.data_ptr() != t.data_ptr()
        with pytest.raises(ValueError, match="16-byte aligned"):
            kv4._rows(t, "out")
    for t in (base[:n].view(2, 4, 3, 128), base[:n].view(2, 3, 4, 128).transpose(1, 2), base[:n].view(2, 4, 3, 128)[..., 64:]):
        assert kv4._rows(t)[0] is t and kv4._rows(t, "out")[0] is t


# ---------------------------------------------------------------- what recorded steps hold
def test_the_evicted_counts_stay_where_a_recorded_step_reads_them(plain_eviction):
    c = filled([90, 70])
    c.evict(40)
    held = c._shifts
    assert held.tolist() == [50, 30]
    c.free(0)
    c.free(1)
    assert c._shifts is held and held.tolist() == [0, 0] and c.evicted == [0, 0]
    c._grow([60, 50])
    c.host_lens = [60, 50]
    c.lens.copy_(torch.tensor([60, 50], dtype=torch.int32))
    c.evict(45)
    assert c._shifts is held and held.tolist() == [15, 5]
    c.set_lengths([0, 45])
    assert c._shifts is held and held.tolist() == [0, 5] and c._next_positions().tolist() == [0, 50]
    c.reset()
    assert c._shifts is None


# ---------------------------------------------------------------- numbers past the kernels' ints
MOST = 2 ** 31 - 1


@pytest.mark.parametrize("fn,base,change,text", [
    # the loops over kept rows and weights step by 1024 from below these: their ints would wrap
    ("nq_select_keys", SELECT, dict(keep=MOST), b"2^30"),
    ("nq_select_keys", SELECT, dict(keep=2 ** 30 + 1), b"2^30"),
    ("nq_select_keys", SELECT, dict(W=MOST), b"2^30"),
    # (len + 31) / 32 steps
    ("nq_attn_decode_kv4", DECODE, dict(max_len=MOST, page=1 << 20, cols=2048, bts=2048, ps=i64(136 << 22, 136 << 20)), b"2^30"),
    ("nq_key_weights", WEIGHTS, dict(max_len=MOST, page=1 << 20, cols=2048, bts=2048), b"2^30"),
])
def test_c_entries_refuse_what_their_ints_cannot_count(fn, base, change, text):
    test_c_entries_refuse(fn, base, change, text)


def big_pool(P=1 << 20):
    """One page of 2^20 rows (torch.empty touches no memory), and a table that names it 8192 times."""
    return kv4.kv4_empty_pool(1, 1, P, 32, device="cpu"), torch.zeros(1, 8192, dtype=torch.int32)


def test_numbers_past_an_int_are_refused(host_calls):
    """ctypes would cut them: row 2^32 + 3 would be stored as row 3."""
    pool, table = big_pool()
    r = rows(H=1, S=1, D=32)
    q = torch.zeros(1, 1, 32, dtype=torch.bfloat16)
    for far in (2 ** 32 + 3, 2 ** 31 - 1):
        with pytest.raises(ValueError, match="outside"):
            kv4.kv4_append(r, r, pool, table, row_offset=far)
        with pytest.raises(ValueError, match="outside"):
            kv4.kv4_gather(pool, table, S=1, row_offset=far)
    with pytest.raises(AssertionError, match="was not refused"):
        kv4.kv4_append(r, r, pool, table, row_offset=2 ** 31 - 2)
    for far in (2 ** 32 + 5, 2 ** 30 + 1):
        with pytest.raises(ValueError, match="max_len"):
            kv4.attention_decode_kv4(q, pool, table, LENS, max_len=far)
        with pytest.raises(ValueError, match="max_len"):
            kv4.attention_key_weights(r, pool, table, LENS, torch.zeros(1, 1, 1), max_len=far)
    with pytest.raises(ValueError, match="2\\^30"):
        kv4.select_keys(torch.zeros(1, 1, 8), LENS, keep=2 ** 30 + 1)
    wide = torch.empty(1, 1, 2 ** 32 + 8, device="meta")
    with pytest.raises(ValueError, match="2\\^30"):
        kv4.select_keys(wide, LENS, keep=8)
    with pytest.raises(ValueError, match="2\\^31"):
        kv4.kv_compact(pool, TABLE, torch.zeros(1, 1, dtype=torch.int32) + 1, torch.zeros(1, 1, 8, dtype=torch.int32), weights=wide)


@pytest.mark.parametrize("name", ["k", "v", "q", "q_weight", "k_weight", "cos", "sin"])
def test_append_refuses_any_operand_that_wants_a_gradient(monkeypatch, name):
    monkeypatch.setattr(kv4.ops, "_require_device", lambda *a: None)
    monkeypatch.setattr(kv4, "_launch", lambda plan, t, fn, args, name, keep, result: result)
    args = dict(k=rows(), v=rows(), q=rows(H=4), q_weight=torch.ones(64), k_weight=torch.ones(64), cos=torch.ones(8, 32),
                sin=torch.ones(8, 32))

    def call(**change):
        a = dict(args, **change)
        return kv4.kv4_append(a.pop("k"), a.pop("v"), pool4(), TABLE, **a)
    leaf = args[name].clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        call(**{name: leaf})
    with pytest.raises(RuntimeError, match="no gradient"):
        call(**{name: torch.nn.Parameter(args[name])})
    with torch.no_grad():
        call(**{name: leaf})
    call(**{name: leaf.detach()})
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        call(**{name: fwd.make_dual(args[name], args[name])})


@pytest.mark.parametrize("shift", [None, LENS])
@pytest.mark.parametrize("change", [dict(position_ids=torch.tensor([[0, 7, 8]])), dict(position_ids=torch.tensor([-1, 0, 1])),
                                    dict(pos_offset=6), dict(pos_offset=-1), dict(pos_offset=2 ** 32)])
def test_positions_outside_the_tables_are_refused_shifted_or_not(host_calls, change, shift):
    tables = dict(cos=torch.ones(8, 32), sin=torch.ones(8, 32))
    with pytest.raises(IndexError):
        kv4.kv4_append(rows(), rows(), pool4(), TABLE, pos_shift=shift, **tables, **change)
    with pytest.raises(AssertionError, match="was not refused"):
        kv4.kv4_append(rows(), rows(), pool4(), TABLE, pos_shift=shift, pos_offset=5, **tables)
    with pytest.raises(AssertionError, match="was not refused"):
        kv4.kv4_append(rows(), rows(), pool4(), TABLE, pos_shift=shift, position_ids=torch.tensor([[7, 0, 3]]), **tables)


@pytest.mark.parametrize("name", ["row_base", "pos_base", "pos_shift"])
def test_lengths_written_over_lengths_read_are_refused(host_calls, name):
    """lens_out as a view that starts among the other's elements: the C entry and the Python call."""
    buf = torch.ones(12, dtype=torch.int32)
    r = rows(B=4)
    table = TABLE.expand(4, 3).contiguous()

    def call(t, out):
        args = {"row_base": buf.new_ones(4), name: t}
        kv4.kv4_append(r, r, pool4(), table, lens_out=out, **args)
    for t, out in ((buf[1:5], buf[4:8]), (buf[4:8], buf[1:5]), (buf[:4], buf[:4])):
        with pytest.raises(ValueError, match="share memory"):
            call(t, out)
    # beside them, or copied before the launch
    for t, out in ((buf[:4], buf[4:8]), (buf[8:], buf[4:8]), (buf[0:8:2], buf[3:7]), (buf[:4].long(), buf[:4])):
        with pytest.raises(AssertionError, match="was not refused"):
            call(t, out)
    at = lambda n: ctypes.c_void_p((1 << 22) + 4 * n)  # noqa: E731
    for t, out in ((at(0), at(1)), (at(1), at(0)), (at(1), at(1))):  # of B = 2
        test_c_entries_refuse("nq_kv4_append", APPEND, {name: t, "lens_out": out}, b"alias")


# ---------------------------------------------------------------- what a failed call leaves behind
def test_growing_takes_all_pages_or_none():
    """A sequence that got its pages before another found none had them in no table: the next
    growth saw nothing to write, and its rows went to page 0."""
    c = nq.PagedKVCache(3, page_size=32, max_pages_per_seq=4)
    c._setup(2, 1, 32, torch.bfloat16, "cpu")
    c._grow([20, 20])
    c.host_lens = [20, 20]
    with pytest.raises(RuntimeError, match="out of pages"):
        c._grow([50, 50])
    assert [len(p) for p in c._pages] == [1, 1] and c.free_pages == 1
    with pytest.raises(ValueError, match="max_pages_per_seq"):
        c._grow([50, 1000])
    assert [len(p) for p in c._pages] == [1, 1] and c.free_pages == 1
    c._grow([50, 20])
    assert c.block_table[0, :2].tolist() == c._pages[0] and len(set(sum(c._pages, []))) == 3


@pytest.mark.parametrize("fails", ["select_keys", "kv_compact"])
@pytest.mark.parametrize("spare", [20, 3])
def test_an_eviction_that_fails_loses_no_pages(plain_eviction, monkeypatch, fails, spare):
    lens = [90, 33, 70, 200]
    used = sum(-(-n // 32) for n in lens)
    c, other = filled(lens, num_pages=used + spare), filled(lens, num_pages=used + spare)
    state = lambda x: (x._free, x._pages, x.host_lens, x.evicted, x.lens.tolist(), x.block_table.tolist())  # noqa: E731
    before = repr(state(c))
    weights = c.weights.clone()

    def out_of_memory(*a, **k):
        raise torch.OutOfMemoryError("no memory")
    with monkeypatch.context() as m:
        m.setattr(attention.kv4, fails, out_of_memory)
        for _ in range(3):
            with pytest.raises(torch.OutOfMemoryError):
                c.evict(40, recent=8)
    assert repr(state(c)) == before and torch.equal(c.weights, weights) and all_pages(c) == list(range(used + spare))
    c.evict(40, recent=8)
    other.evict(40, recent=8)
    assert repr(state(c)) == repr(state(other)) and torch.equal(c.weights, other.weights)
    assert all_pages(c) == list(range(used + spare))


def stub_forward(monkeypatch, max_pos=1024):
    """An Attention whose kernels do nothing: a call of _paged_forward on host tensors."""
    attn = nq.Attention(nq.AttentionConfig(hidden_size=64, num_attention_heads=2, num_key_value_heads=1, head_dim=32,
                                           max_position_embeddings=max_pos))
    monkeypatch.setattr(attention.ops, "kv_append_paged", lambda *a, **k: None)
    monkeypatch.setattr(attention.ops, "attention_prefill_paged", lambda q, *a, **k: q)
    monkeypatch.setattr(attention.ops, "attention_decode_paged",
                        lambda q, kp, vp, table, lens, *, lens_out, **k: (lens_out.copy_(lens + 1), q)[1])
    attn.o_proj = torch.nn.Identity()

    def forward(cache, S):
        q, k, v = (torch.zeros(2, h, S, 32, dtype=torch.bfloat16) for h in (2, 1, 1))
        with torch.no_grad():
            attn._paged_forward(q, k, v, None, cache, None, None, None, None, 1e-6)
    return forward


def test_expected_lengths_wait_for_the_next_longer_forward(monkeypatch):
    """Neither a one-token forward nor one that cannot run uses them up."""
    forward = stub_forward(monkeypatch)
    c = nq.PagedKVCache(6, page_size=32, max_pages_per_seq=8)
    forward(c, 3)
    c.expect_lengths([5, 20])
    forward(c, 1)
    assert c.host_lens == [4, 4]
    with pytest.raises(RuntimeError, match="out of pages"):
        forward(c, 100)
    with pytest.raises(IndexError):
        forward(c, 2000)
    assert c.host_lens == [4, 4] == c.lens.tolist()
    forward(c, 20)
    assert c.host_lens == [9, 24] == c.lens.tolist()
    c.set_lengths([9, 9])
    forward(c, 2)
    assert c.host_lens == [11, 11]  # asked for once
    c.expect_lengths([1, 3])
    with pytest.raises(ValueError, match="do not fit"):
        forward(c, 2)
    assert c.host_lens == [11, 11] == c.lens.tolist()


def test_queries_far_apart_are_copied(monkeypatch):
    """The last queries of a long prompt lie as far apart as the prompt's heads do; the kernel
    addresses 256 rows with 32-bit offsets."""
    seen = []
    monkeypatch.setattr(kv4, "_check", lambda *a: None)
    monkeypatch.setattr(kv4, "_launch", lambda plan, t, fn, args, name, keep, result: seen.append((args, keep[0])) or result)
    base = torch.empty(2 ** 30 + 2 ** 27, dtype=torch.bfloat16)  # touched at a few rows only

    def call(q):
        kv4.attention_key_weights(q, pool4(D=32, H=1), TABLE, LENS, torch.zeros(q.shape[:3]), max_len=90)
        args, kept = seen.pop()
        assert args[0] == kept.data_ptr() and list(args[1]) == list(kept.stride()[:3])
        return kept
    head = 2 ** 29 + 8
    far = base.as_strided((1, 2, 3, 32), (0, head, 64, 1))
    for h in range(2):
        for s in range(3):
            far[0, h, s] = torch.arange(32) + 100 * h + 10 * s
    got = call(far)
    assert torch.equal(got, far) and got.stride()[1:] == (32, 64, 1)
    got = call(base.as_strided((1, 2, 3, 32), (0, 32, 2 ** 29, 1)))
    assert got.stride()[1:] == (32, 64, 1)
    near = base.as_strided((1, 2, 3, 32), (0, 2 ** 29, 64, 1))
    assert call(near) is near
