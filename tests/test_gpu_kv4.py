"""4-bit pages on the GPU: rows stored and read back, attention over them, key weights,
selection and compaction, each against its definition in 64 bits (tests/kv4_reference.py)."""

import math

import pytest
import torch

import nano_qwen_amd as nq
from oracle import rope_tables
from tests import kv4_reference as ref
from tests.helpers import say

pytestmark = pytest.mark.gpu
DEV = "cuda"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(*shape, g, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def table_for(lens, P, g, spare=3, cols=None):
    """(block table, pages): pages in no order; entries behind a sequence's are no pages."""
    need = [-(-n // P) for n in lens]
    pages = sum(need) + spare
    ids = torch.randperm(pages, generator=g, device=DEV).int()
    table = torch.full((len(lens), cols or max(max(need), 1)), 2 ** 30, dtype=torch.int32, device=DEV)
    at = 0
    for b, m in enumerate(need):
        table[b, :m] = ids[at:at + m]
        at += m
    return table, pages


def random_pool(pages, H, P, D, g):
    pool = nq.kv4_empty_pool(pages, H, P, D, DEV)
    ref.fill_pool(pool, randn(pages, H, P, D, g=g), randn(pages, H, P, D, g=g))
    return pool


def pool_values(pool):
    return [ref.values(*x) for x in ref.read_pool(pool)]


# ---------------------------------------------------------------- rows

EDGES = [0.0, -0.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, -0.25, -1.25, -5.0, 0.2499, 0.7501]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,P,B,H,S", [(128, 64, 2, 4, 77), (64, 32, 3, 1, 33), (32, 96, 1, 2, 1), (128, 32, 1, 8, 200)])
def test_rows_are_stored_as_defined_and_read_back(D, P, B, H, S, dtype):
    say(f"rows D{D} P{P} B{B} H{H} S{S} {dtype}")
    g = gen(D + S)
    k, v = (randn(B, S, H, D, g=g) * torch.exp(3 * randn(B, S, H, 1, g=g)) for _ in range(2))
    edges = torch.tensor(EDGES, device=DEV)
    k[0, 0, 0, :16] = edges * 2.0 ** 5
    k[0, 0, 0, 16:32] = -edges
    v[0, 0, 0, :32] = 0.0
    v[-1, -1, -1, :32] = torch.linspace(-7, 7, 32, device=DEV) * 2.0 ** -20
    k, v = k.to(dtype).transpose(1, 2), v.to(dtype).transpose(1, 2)
    row0 = 13
    table, pages = table_for([row0 + S] * B, P, g)
    pool = nq.kv4_empty_pool(pages, H, P, D, DEV)
    pool.fill_(77)
    before = pool.clone()
    nq.kv4_append(k, v, pool, table, row_offset=row0)
    for x, (codes, byte) in zip((k, v), ref.read_pool(pool)):
        want_codes, want_byte = ref.quantise(x)
        for b in range(B):
            got = ref.rows_of(codes, table[b], row0 + S)[:, row0:]
            assert torch.equal(got, want_codes[b])
            assert torch.equal(ref.rows_of(byte, table[b], row0 + S)[:, row0:], want_byte[b])
    # rows that are not the call's keep what they held
    fresh = before.clone()
    nq.kv4_append(k, v, fresh, table, row_offset=row0)
    for a, b_, new in zip(ref.parts(before), ref.parts(pool), ref.parts(fresh)):
        for b in range(B):
            assert torch.equal(ref.rows_of(a, table[b], row0), ref.rows_of(b_, table[b], row0))
    used = torch.unique(table[table < pages]).long()
    untouched = torch.ones(pages, dtype=torch.bool, device=DEV)
    untouched[used] = False
    assert torch.equal(pool[untouched], before[untouched])
    for out in (torch.bfloat16, torch.float32):
        kr, vr = nq.kv4_gather(pool, table, S=S, row_offset=row0, dtype=out)
        assert torch.equal(kr.double(), ref.stored(k)) and torch.equal(vr.double(), ref.stored(v))


def test_extreme_rows():
    """Denormal, huge, infinite and NaN elements; zeros."""
    say("extreme rows")
    g = gen(3)
    x = torch.zeros(1, 1, 8, 64, device=DEV)
    x[0, 0, 0] = 2.0 ** -140 * torch.arange(64, device=DEV)
    x[0, 0, 1] = 2.0 ** -126 * torch.linspace(-9, 9, 64, device=DEV)
    x[0, 0, 2] = 3.3e38 * torch.linspace(-1, 1, 64, device=DEV)
    x[0, 0, 3] = randn(64, g=g)
    x[0, 0, 3, 5] = math.inf
    x[0, 0, 4] = randn(64, g=g)
    x[0, 0, 4, 40] = math.nan
    x[0, 0, 5] = 2.0 ** 127
    x[0, 0, 6] = 1.75 * 2.0 ** 10
    x[0, 0, 6, 1] = torch.nextafter(torch.tensor(1.75 * 2.0 ** 10), torch.tensor(1e9))
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    pool = nq.kv4_empty_pool(1, 1, 32, 64, DEV)
    nq.kv4_append(x, x.flip(2).contiguous(), pool, table)
    (codes, byte), _ = ref.read_pool(pool)
    want_codes, want_byte = ref.quantise(x)
    assert torch.equal(byte[0, :, :8], want_byte[0])
    ok = (want_byte != 255).repeat_interleave(32, -1)
    assert torch.equal(codes[0, :, :8][ok[0]], want_codes[0][ok[0]])
    k, _ = nq.kv4_gather(pool, table, S=8, dtype=torch.float32)
    want = ref.stored(x)
    assert torch.equal(torch.isnan(k), torch.isnan(want))
    assert torch.equal(k.double()[~torch.isnan(want)], want[~torch.isnan(want)])


@pytest.mark.parametrize("wdtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_norm_and_rotation_match_the_row_kernel(D, dtype, wdtype):
    """K rows are quantised from the very fp32 rows that the row kernel forms; q rows are its."""
    if wdtype == torch.bfloat16 and dtype != torch.bfloat16:
        pytest.skip("bf16 weights go with bf16 rows")
    say(f"norm and rotation D{D} {dtype} {wdtype}")
    g = gen(D)
    B, Hq, H, S, P = 3, 6, 2, 5, 32
    k, v = (randn(B, S, H, D, g=g, dtype=dtype).transpose(1, 2) for _ in range(2))
    q = randn(B, S, Hq, D, g=g, dtype=dtype).transpose(1, 2)
    kw, qw = ((1 + 0.1 * randn(D, g=g)).to(wdtype) for _ in range(2))
    cos, sin = (t.to(DEV) for t in rope_tables(D, 512, 10000.0))
    lens = torch.tensor([0, 17, 63], dtype=torch.int32, device=DEV)
    shift = torch.tensor([0, 5, 100], dtype=torch.int32, device=DEV)
    table, pages = table_for([n + S for n in (0, 17, 63)], P, g)
    pool = nq.kv4_empty_pool(pages, H, P, D, DEV)
    lens_out = torch.empty_like(lens)
    q_hat = nq.kv4_append(k, v, pool, table, q=q, q_weight=qw, k_weight=kw, cos=cos, sin=sin, pos_base=lens,
                          pos_shift=shift, row_base=lens, lens_out=lens_out)
    assert torch.equal(lens_out, lens + S)
    k32 = torch.empty(B, H, S, D, device=DEV)
    nq.qk_norm_rope(k=k, k_out=k32, k_weight=kw, cos=cos, sin=sin, pos_base=lens + shift)
    q_want, _, _ = nq.qk_norm_rope(q=q, q_weight=qw, cos=cos, sin=sin, pos_base=lens + shift)
    assert torch.equal(q_hat, q_want)
    kr, vr = nq.kv4_gather(pool, table, S=S, row_base=lens, dtype=torch.float32)
    assert torch.equal(kr.double(), ref.stored(k32)) and torch.equal(vr.double(), ref.stored(v))


def test_sequences_that_do_not_fit_store_nothing():
    say("lengths and pages out of range")
    g = gen(5)
    H, D, P = 2, 64, 32
    k, v = (randn(4, H, 3, D, g=g) for _ in range(2))
    table = torch.tensor([[0, 1], [2, 3], [4, 99], [-5, 5]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([-1, 62, 31, 31], dtype=torch.int32, device=DEV)
    pool = nq.kv4_empty_pool(6, H, P, D, DEV)
    pool.zero_()
    lens_out = torch.empty_like(lens)
    nq.kv4_append(k, v, pool, table, row_base=lens, lens_out=lens_out)
    assert lens_out.tolist() == [-1, 62, 34, 34]
    assert int(pool[:4].long().sum()) == 0  # sequences 0 and 1
    kr, _ = nq.kv4_gather(pool, table, S=3, row_base=lens, dtype=torch.float32)
    want = ref.stored(k)
    assert torch.isnan(kr[0, :, 0]).all() and torch.isnan(kr[1, :, 2]).all()
    assert torch.equal(kr[2, :, 0].double(), want[2, :, 0]) and torch.isnan(kr[2, :, 1:]).all()
    assert torch.isnan(kr[3, :, 0]).all() and torch.equal(kr[3, :, 1:].double(), want[3, :, 1:])


# ---------------------------------------------------------------- decode

def decode_bound(dtype, out, mass, spread, n, D):
    """How far an output may lie from the definition's.

    bf16: the probabilities round to bf16 (2^-8 relative each, in the numerator), and the
    output.  Both types: a score is a sum of D products in fp32 (2^-24 each, of at most
    `spread` together; the hardware's inner sums may drop the bits below, so twice), it
    enters an exponential together with an fp32 multiply and one more rounding of as large
    a number; the sums over n keys and their partials round n + 64 times.  fp32: three bf16
    terms hold 24 bits of a probability and of q.
    """
    u = 2.0 ** -24
    rel = spread[:, None] * (2 * D + 8) * u * 2 + (n + 64) * u + 2.0 ** -21
    tol = mass * rel
    if dtype == torch.bfloat16:
        tol = tol + mass * 2.0 ** -8 + (out.abs() + mass * 2.0 ** -8) * 2.0 ** -8
    return tol


def check_decode(o, lse, q, pool, table, lens, P, what):
    kv, vv = pool_values(pool)
    D = q.shape[-1]
    scale = 1 / math.sqrt(D)
    for b, n in enumerate(lens):
        if n == 0:
            assert (o[b] == 0).all() and (lse[b] == -math.inf).all()
            continue
        want, want_lse, mass, spread = ref.attention(q[b], ref.rows_of(kv, table[b], n), ref.rows_of(vv, table[b], n), scale)
        tol = decode_bound(q.dtype, want, mass, spread, n, D)
        err = (o[b].double() - want).abs()
        assert (err <= tol).all(), f"{what} b={b}: {float((err / tol).max()):.3f} of the bound, {float(err.max()):.3e}"
        lse_tol = spread * (2 * D + 8) * 2.0 ** -23 + (want_lse.abs() + 1) * 2.0 ** -20 + (n + 64) * 2.0 ** -24
        assert ((lse[b].double() - want_lse).abs() <= lse_tol).all(), what


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,Hq,Hkv,D,P,lens", [
    (1, 8, 8, 128, 64, [1]),
    (1, 16, 8, 128, 64, [512]),
    (3, 4, 2, 128, 32, [1, 0, 33]),
    (4, 14, 2, 64, 96, [97, 1500, 31, 32]),
    (2, 17, 1, 128, 64, [700, 64]),
    (2, 64, 2, 64, 32, [65, 2049]),
    (5, 3, 1, 32, 32, [5, 63, 64, 999, 0]),
    (1, 32, 2, 32, 128, [5000]),
    (70, 2, 1, 64, 32, [(37 * i) % 200 for i in range(70)]),
    (1, 5, 1, 128, 32, [40000]),
    (12, 64, 4, 128, 64, [3000 + 317 * i for i in range(12)]),
])
def test_decode(B, Hq, Hkv, D, P, lens, dtype):
    say(f"decode B{B} {Hq}/{Hkv} D{D} P{P} {dtype}")
    g = gen(sum(lens) + Hq)
    table, pages = table_for(lens, P, g)
    pool = random_pool(pages, Hkv, P, D, g)
    # what lies behind a sequence's last key must not matter: NaN blocks
    _, _, ks, vs = ref.parts(pool)
    for b, n in enumerate(lens):
        if n % P:
            last = int(table[b, n // P])
            ks[last, :, n % P:] = 255
            vs[last, :, n % P:] = 255
    q = randn(B, Hq, D, g=g, dtype=dtype)
    lens_t = torch.tensor(lens, dtype=torch.int32, device=DEV)
    o, lse = nq.attention_decode_kv4(q, pool, table, lens_t, max_len=max(lens) if max(lens) else 1, return_lse=True)
    check_decode(o, lse, q, pool, table, lens, P, f"decode {dtype}")
    again = nq.attention_decode_kv4(q, pool, table, lens_t, max_len=max(lens))
    assert torch.equal(o, again)


def test_decode_of_lengths_and_pages_out_of_range():
    say("decode: lengths and pages out of range")
    g = gen(11)
    table, pages = table_for([100, 100, 100, 100], 32, g)
    pool = random_pool(pages, 2, 32, 64, g)
    q = randn(4, 4, 64, g=g, dtype=torch.bfloat16)
    lens = torch.tensor([-1, 101, 100, 100], dtype=torch.int32, device=DEV)
    table[3, 1] = pages
    o, lse = nq.attention_decode_kv4(q, pool, table, lens, max_len=100, return_lse=True)
    assert torch.isnan(o[[0, 1, 3]]).all() and torch.isnan(lse[[0, 1, 3]]).all()
    check_decode(o[2:3], lse[2:3], q[2:3], pool, table[2:3], [100], 32, "the sequence beside them")


def test_nan_block_reaches_only_its_own_sequence_and_head():
    say("decode: NaN blocks")
    g = gen(12)
    table, pages = table_for([64, 64], 32, g)
    pool = random_pool(pages, 2, 32, 128, g)
    _, _, ks, vs = ref.parts(pool)
    ks[int(table[0, 0]), 1, 3, 2] = 255
    q = randn(2, 4, 128, g=g, dtype=torch.bfloat16)
    lens = torch.tensor([64, 64], dtype=torch.int32, device=DEV)
    o = nq.attention_decode_kv4(q, pool, table, lens, max_len=64)
    assert torch.isnan(o[0, 2:]).all() and torch.isfinite(o[0, :2]).all() and torch.isfinite(o[1]).all()
    ks[int(table[0, 0]), 1, 3, 2] = 120
    vs[int(table[1, 1]), 0, 9, 1] = 255  # one block of a value row: its 32 output elements
    o = nq.attention_decode_kv4(q, pool, table, lens, max_len=64)
    assert torch.isnan(o[1, :2, 32:64]).all() and torch.isfinite(o[1, :2, :32]).all() and torch.isfinite(o[1, :2, 64:]).all()
    assert torch.isfinite(o[0]).all() and torch.isfinite(o[1, 2:]).all()


def test_strides_scale_and_types_of_tables():
    say("decode: strides, scale, int64 tables")
    g = gen(13)
    lens = [77, 130]
    table, pages = table_for(lens, 32, g, cols=9)
    big = torch.zeros(pages, 3, 32, 136, dtype=torch.uint8, device=DEV)
    pool = big[:, 1:3]
    ref.fill_pool(pool, randn(pages, 2, 32, 128, g=g), randn(pages, 2, 32, 128, g=g))
    wide = randn(2, 8, 3, 128, g=g, dtype=torch.bfloat16)
    q = wide[:, ::2, 1]
    out = torch.zeros(2, 4, 2, 128, dtype=torch.bfloat16, device=DEV)
    lens_t = torch.tensor(lens, device=DEV)
    nq.attention_decode_kv4(q, pool, table.long(), lens_t, max_len=130, sm_scale=0.05, out=out[:, :, 1])
    assert (out[:, :, 0] == 0).all()
    kv, vv = pool_values(pool)
    for b, n in enumerate(lens):
        want, _, mass, spread = ref.attention(q[b], ref.rows_of(kv, table[b], n), ref.rows_of(vv, table[b], n), 0.05)
        assert ((out[b, :, 1].double() - want).abs() <= decode_bound(q.dtype, want, mass, spread, n, 128)).all()


# ---------------------------------------------------------------- key weights

def weights_case(B, Hq, Hkv, D, P, S, lens, four, seed):
    g = gen(seed)
    table, pages = table_for(lens, P, g)
    if four:
        pool = random_pool(pages, Hkv, P, D, g)
        kv = pool_values(pool)[0]
    else:
        pool = randn(pages, Hkv, P, D, g=g, dtype=torch.bfloat16)
        kv = pool.double()
    q = randn(B, S, Hq, D, g=g, dtype=torch.bfloat16).transpose(1, 2)
    scale = 1 / math.sqrt(D)
    lse = torch.full((B, Hq, S), -math.inf, dtype=torch.float32, device=DEV)
    for b, n in enumerate(lens):
        k = ref.rows_of(kv, table[b], n)
        s = (q[b].double().reshape(Hkv, -1, D) @ k.transpose(1, 2).contiguous() * scale).view(Hq, S, n)
        if S > 1:
            s = s.masked_fill(~torch.ones(S, n, dtype=torch.bool, device=DEV).tril(n - S), -math.inf)
        lse[b] = torch.logsumexp(s, -1).float()
    return q, pool, table, kv, lse, scale


def check_weights(w, q, kv, table, lens, lse, scale, causal=True, base=None):
    B, Hq, S, D = q.shape
    for b, n in enumerate(lens):
        k = ref.rows_of(kv, table[b], n)
        want = ref.key_weights(q[b], k, lse[b], scale, causal)
        spread = 0.0
        if n:
            spread = float((q[b].double().abs().reshape(kv.shape[1], -1, D) @ k.abs().transpose(1, 2).contiguous()).max()) * scale
        # a score as in decode_bound, and lse's fp32 times log2 e
        top = float(torch.where(torch.isfinite(lse[b]), lse[b].abs(), 0.0).max())
        rel = (spread * (2 * D + 8) + 4 * top + Hq // kv.shape[1] * S + 16) * 2.0 ** -23
        old = 0.0 if base is None else base[b, :, :n].double()
        tol = want * rel + 1e-37 + (0 if base is None else 2.0 ** -24 * (want + old))
        err = (w[b, :, :n].double() - old - want).abs()
        assert (err <= tol).all(), f"b={b}: {float((err / tol).max())}"
        rest = w[b, :, n:]
        assert (rest == 0).all() if base is None else torch.equal(rest, base[b, :, n:])


@pytest.mark.parametrize("four", [True, False])
@pytest.mark.parametrize("B,Hq,Hkv,D,P,S,lens", [
    (1, 8, 8, 128, 64, 1, [1]),
    (3, 16, 2, 128, 32, 1, [300, 0, 65]),
    (2, 40, 2, 64, 96, 1, [1000, 64]),
    (2, 6, 2, 32, 32, 7, [40, 7]),
    (1, 4, 1, 128, 64, 100, [612]),
    (2, 4, 4, 64, 32, 257, [257, 300]),
    (1, 5, 1, 128, 32, 33, [2000]),
    (2, 16, 2, 64, 64, 300, [1700, 301]),
    (1, 64, 2, 32, 32, 600, [900]),
])
def test_key_weights(B, Hq, Hkv, D, P, S, lens, four):
    say(f"key weights B{B} {Hq}/{Hkv} D{D} P{P} S{S} four={four}")
    q, pool, table, kv, lse, scale = weights_case(B, Hq, Hkv, D, P, S, lens, four, sum(lens) + S)
    lens_t = torch.tensor(lens, dtype=torch.int32, device=DEV)
    top = max(max(lens), 1)
    w = nq.attention_key_weights(q, pool, table, lens_t, lse, max_len=top)
    assert w.shape == (B, Hkv, top)
    check_weights(w, q, kv, table, lens, lse, scale)
    assert torch.equal(w, nq.attention_key_weights(q, pool, table, lens_t, lse, max_len=top))
    # each query's weights sum to one
    if all(n >= S for n in lens):
        total = w.double().sum(-1)
        assert torch.allclose(total, torch.full_like(total, Hq // Hkv * S), rtol=1e-4)
    base = torch.rand(B, Hkv, top + 5, device=DEV)
    acc = base.clone()
    assert nq.attention_key_weights(q, pool, table, lens_t, lse, max_len=top, weights=acc) is acc
    check_weights(acc, q, kv, table, lens, lse, scale, base=base)
    full = nq.attention_key_weights(q, pool, table, lens_t, lse, max_len=top, causal=False)
    check_weights(full, q, kv, table, lens, lse, scale, causal=False)


def test_key_weights_of_more_queries_than_keys_and_bad_lengths():
    say("key weights: odd lengths")
    q, pool, table, kv, lse, scale = weights_case(3, 4, 2, 64, 32, 9, [5, 40, 40], True, 5)
    assert (lse[0, :, :4] == -math.inf).all()
    lens = torch.tensor([5, -3, 41], dtype=torch.int32, device=DEV)
    w = nq.attention_key_weights(q, pool, table, lens, lse, max_len=40)
    check_weights(w[:1], q[:1], kv, table[:1], [5], lse[:1], scale)
    assert torch.isnan(w[1:]).all()
    lens = torch.tensor([5, 40, 40], dtype=torch.int32, device=DEV)
    table[2, 1] = -1
    w = nq.attention_key_weights(q, pool, table, lens, lse, max_len=40)
    check_weights(w[1:2], q[1:2], kv, table[1:2], [40], lse[1:2], scale)
    assert torch.isnan(w[2, :, 32:]).all() and torch.isfinite(w[2, :, :32]).all()


@pytest.mark.parametrize("four", [True, False])
def test_key_weights_of_several_runs_a_wave(four):
    """Enough keys for waves of two, three and four runs, and last waves of one."""
    for B, Hkv, top in ((130, 8, 1030), (200, 8, 1030), (300, 8, 1000)):
        say(f"key weights: {B} sequences of up to {top} keys, four={four}")
        lens = [(37 * i * i + 61) % (top + 1) for i in range(B - 1)] + [top]
        q, pool, table, kv, lse, scale = weights_case(B, 2 * Hkv, Hkv, 32, 32, 1, lens, four, B)
        lens_t = torch.tensor(lens, dtype=torch.int32, device=DEV)
        w = nq.attention_key_weights(q, pool, table, lens_t, lse, max_len=top)
        base = torch.rand(B, Hkv, top, device=DEV)
        acc = nq.attention_key_weights(q, pool, table, lens_t, lse, max_len=top, weights=base.clone())
        some = list(range(0, B, 9)) + [B - 1]
        pick = lambda x: x[some]  # noqa: E731
        check_weights(pick(w), pick(q), kv, pick(table), [lens[b] for b in some], pick(lse), scale)
        check_weights(pick(acc), pick(q), kv, pick(table), [lens[b] for b in some], pick(lse), scale, base=pick(base))


@pytest.mark.parametrize("causal", [True, False])
def test_key_weights_of_many_chunks_of_rows(causal):
    say(f"key weights: 75 chunks of rows, three ranges of keys, causal={causal}")
    q, pool, table, kv, lse, scale = weights_case(1, 32, 1, 32, 32, 600, [2500], True, 77)
    w = nq.attention_key_weights(q, pool, table, torch.tensor([2500], device=DEV), lse, max_len=2500, causal=causal)
    check_weights(w, q, kv, table, [2500], lse, scale, causal=causal)


@pytest.mark.parametrize("four", [True, False])
@pytest.mark.parametrize("S,Hq", [(1, 4), (3, 4), (40, 4), (300, 6), (65, 4)])
def test_queries_that_saw_nothing_add_nothing(S, Hq, four):
    """Whatever they hold: NaN behind a padded sequence's last query, infinities."""
    say(f"key weights: unused queries S{S} four={four}")
    q, pool, table, kv, lse, scale = weights_case(2, Hq, 2, 64, 32, S, [400, 350], four, S)
    lens = torch.tensor([400, 350], dtype=torch.int32, device=DEV)
    q = q.clone()
    lse[1, :, -1] = -math.inf
    lse[0, 1, S // 2] = -math.inf
    want = nq.attention_key_weights(q, pool, table, lens, lse, max_len=400)
    q[1, :, -1] = math.nan
    q[0, 1, S // 2] = math.inf
    got = nq.attention_key_weights(q, pool, table, lens, lse, max_len=400)
    assert torch.isfinite(got).all() and torch.equal(got, want)
    q[0, 2, S - 1] = math.nan  # of one that saw keys: theirs are NaN, the other head's and sequence's are not
    got = nq.attention_key_weights(q, pool, table, lens, lse, max_len=400)
    assert torch.isnan(got[0, 2 // (Hq // 2)]).any() and torch.equal(got[0, 1 - 2 // (Hq // 2)], want[0, 1 - 2 // (Hq // 2)])
    assert torch.equal(got[1], want[1])


# ---------------------------------------------------------------- eviction

@pytest.mark.parametrize("lens,keep,recent,first", [
    ([10], 4, 1, 1), ([1], 1, 0, 0), ([100, 3, 0], 50, 10, 4), ([2049, 2000], 700, 0, 0), ([5000], 4999, 64, 4),
    ([70000, 64000], 1000, 1000, 0), ([66000], 30000, 1, 3), ([333], 100, 60, 40),
])
@pytest.mark.parametrize("values", ["spread", "ties", "odd"])
def test_select_keys(lens, keep, recent, first, values):
    say(f"select {lens} keep {keep} recent {recent} first {first} {values}")
    g = gen(keep + len(lens))
    B, H, W = len(lens), 3, max(lens) + 2
    if values == "spread":
        w = torch.exp(3 * randn(B, H, W, g=g))
    elif values == "ties":
        w = torch.randint(0, 4, (B, H, W), generator=g, device=DEV).float() / 8
    else:
        w = randn(B, H, W, g=g)
        for i, x in enumerate((math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-42)):
            w[..., i::11] = x
    lens_t = torch.tensor(lens, dtype=torch.int32, device=DEV)
    kept = nq.select_keys(w, lens_t, keep=keep, recent=recent, first=first)
    host = w.cpu()
    for b, n in enumerate(lens):
        for h in range(H):
            assert kept[b, h].tolist() == ref.select(host[b, h], n, keep, recent, first), (b, h)


def test_select_keys_of_strided_weights_and_bad_lengths():
    say("select: strides, lengths")
    w = torch.rand(3, 4, 100, device=DEV)
    lens = torch.tensor([90, -1, 101], dtype=torch.int32, device=DEV)
    kept = nq.select_keys(w.transpose(0, 1)[:3].transpose(0, 1)[:, 1:], lens, keep=20)
    for h in range(2):
        assert kept[0, h].tolist() == ref.select(w[0, 1 + h].cpu(), 90, 20, 0, 0)
    assert (kept[1:] == -1).all()


@pytest.mark.parametrize("kind", ["four", "bf16", "f32"])
@pytest.mark.parametrize("D,P,H,lens,keep", [(128, 64, 2, [200, 90], 100), (64, 32, 1, [65], 33), (32, 96, 3, [100, 7, 50], 40)])
def test_compact(D, P, H, lens, keep, kind):
    say(f"compact {kind} D{D} P{P} {lens} keep {keep}")
    g = gen(D + keep)
    B, W = len(lens), max(lens) + 3
    new_cols = -(-keep // P) + 1
    table, pages = table_for(lens, P, g, spare=B * new_cols)
    used = set(table[table < pages].tolist())
    new = torch.tensor([i for i in range(pages) if i not in used], dtype=torch.int32, device=DEV)[:B * new_cols].view(B, -1)
    if kind == "four":
        pool = torch.randint(0, 256, (pages, H, P, 17 * D // 16), generator=g, device=DEV, dtype=torch.uint8)
        pools, views = pool, ref.parts(pool)
    else:
        dt = torch.bfloat16 if kind == "bf16" else torch.float32
        pools = tuple(randn(pages, H, P, D, g=g, dtype=dt) for _ in range(2))
        views = list(pools)
    before = [x.clone() for x in views]
    w = torch.rand(B, H, W, generator=g, device=DEV)
    lens_t = torch.tensor(lens, dtype=torch.int32, device=DEV)
    kept = nq.select_keys(w, lens_t, keep=keep, recent=3, first=1)
    out = nq.kv_compact(pools, table, new, kept, weights=w)
    wipe = [x.clone() for x in before]
    for b in range(B):
        for h in range(H):
            for i, j in enumerate(kept[b, h].tolist()):
                if j < 0:
                    assert float(out[b, h, i]) == 0
                    continue
                assert float(out[b, h, i]) == float(w[b, h, j])
                for x, old in zip(wipe, before):
                    x[int(new[b, i // P]), h, i % P] = old[int(table[b, j // P]), h, j % P]
    assert (out[..., keep:] == 0).all()
    for x, want in zip(views, wipe):
        assert torch.equal(x.view(torch.uint8) if x.is_contiguous() else x, want.view(torch.uint8) if x.is_contiguous() else want)


def test_compact_skips_what_is_no_row_or_page():
    say("compact: indices and pages out of range")
    pool = torch.zeros(4, 1, 32, 64, device=DEV)
    v = torch.arange(4 * 32 * 64, device=DEV).float().view(4, 1, 32, 64)
    table = torch.tensor([[0, 77]], dtype=torch.int32, device=DEV)
    new = torch.tensor([[2, 9]], dtype=torch.int32, device=DEV)
    kept = torch.tensor([[[5, 40, 9999, -7] + [1] * 36]], dtype=torch.int32, device=DEV)
    want = v.clone()
    want[2, 0, 0] = v[0, 0, 5]
    want[2, 0, 4:32] = v[0, 0, 1]
    nq.kv_compact((pool, v), table, new, kept)
    assert torch.equal(v, want)


# ---------------------------------------------------------------- large pools

def far(pool, table, pages, n):
    """The pool's pages as the last ones of a pool of n, and the table for them."""
    big = torch.empty(n, *pool.shape[1:], dtype=pool.dtype, device=DEV)
    big[n - pages:] = pool
    return big, torch.where(table < pages, table + (n - pages), table)


@pytest.mark.parametrize("four", [True, False])
def test_pages_past_4_gib(four):
    say(f"pages past 4 GiB, four={four}")
    g = gen(31)
    lens, P, H, D = [300, 129], 64, 8, 128
    table, pages = table_for(lens, P, g, spare=4)
    used = set(table[table < pages].tolist())
    new = torch.tensor([i for i in range(pages) if i not in used], dtype=torch.int32, device=DEV).view(2, 2)
    lens_t = torch.tensor(lens, dtype=torch.int32, device=DEV)
    q = randn(2, 16, D, g=g, dtype=torch.bfloat16)
    lse = torch.full((2, 16), 3.0, device=DEV)
    w = torch.rand(2, H, 320, generator=g, device=DEV)
    kept = nq.select_keys(w, lens_t, keep=100, recent=5)
    if four:
        pool = random_pool(pages, H, P, D, g)
        big, there = far(pool, table, pages, 66000)
        assert big[-pages:].data_ptr() - big.data_ptr() > 2 ** 32
        for S in (1, 40):
            rows = [randn(2, H, S, D, g=g, dtype=torch.bfloat16) for _ in range(2)]
            base = lens_t - S
            nq.kv4_append(*rows, pool, table, row_base=base)
            nq.kv4_append(*rows, big, there, row_base=base)
            assert torch.equal(big[-pages:], pool)
        for x, y in zip(nq.kv4_gather(pool, table, S=129), nq.kv4_gather(big, there, S=129)):
            assert torch.equal(x, y)
        assert torch.equal(nq.attention_decode_kv4(q, pool, table, lens_t, max_len=300),
                           nq.attention_decode_kv4(q, big, there, lens_t, max_len=300))
        keys, far_keys, pools, far_pools = pool, big, pool, big
    else:
        pools = tuple(randn(pages, H, P, D, g=g, dtype=torch.bfloat16) for _ in range(2))
        (keys, values), (far_keys, far_values) = pools, (far(x, table, pages, 33000)[0] for x in pools)
        there = far(keys[:, :1, :1], table, pages, 33000)[1]
        far_pools = (far_keys, far_values)
        assert far_keys[-pages:].data_ptr() - far_keys.data_ptr() > 2 ** 32
    for S in (1, 20, 200):
        qs = randn(2, 16, S, D, g=g, dtype=torch.bfloat16)
        ls = lse[:, :, None].expand(2, 16, S).contiguous()
        assert torch.equal(nq.attention_key_weights(qs, keys, table, lens_t, ls, max_len=300),
                           nq.attention_key_weights(qs, far_keys, there, lens_t, ls, max_len=300))
    n = far_keys.shape[0]
    nq.kv_compact(pools, table, new, kept)
    nq.kv_compact(far_pools, there, new + (n - pages), kept)
    for x, y in ([(pools, far_pools)] if four else zip(pools, far_pools)):
        assert torch.equal(y[-pages:], x)


# ---------------------------------------------------------------- together

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_lse_of_the_plain_paged_decode(dtype):
    say(f"paged decode with lse {dtype}")
    g = gen(21)
    for lens, Hq in (([70, 0, 500], 6), ([9000], 4), ([33], 40)):
        table, pages = table_for(lens, 32, g)
        table = table.clamp(max=pages - 1)
        k, v = (randn(pages, 2, 32, 64, g=g, dtype=dtype) for _ in range(2))
        q = randn(len(lens), Hq, 64, g=g, dtype=dtype)
        lens_t = torch.tensor(lens, dtype=torch.int32, device=DEV)
        kw = dict(max_len=max(lens))
        if dtype == torch.float32 and 128 % (Hq // 2):
            continue
        plain = nq.attention_decode_paged(q, k, v, table, lens_t, **kw)
        o, lse = nq.attention_decode_paged(q, k, v, table, lens_t, return_lse=True, **kw)
        assert torch.equal(o, plain)
        for b, n in enumerate(lens):
            if n == 0:
                assert (lse[b] == -math.inf).all()
                continue
            _, want, _, spread = ref.attention(q[b], ref.rows_of(k, table[b], n).double(), ref.rows_of(v, table[b], n).double(), 1 / 8)
            # the bf16 decode rounds nothing on the way to a score of plain q and k
            tol = spread * (2 * 64 + 8) * 2.0 ** -23 + (want.abs() + 1) * 2.0 ** -20 + (n + 64) * 2.0 ** -24
            assert ((lse[b].double() - want).abs() <= tol).all()


def test_captured_steps_replay():
    """Append, decode, key weights, selection and compaction in one graph, replayed over new
    inputs with eager calls of the same operators in between."""
    say("graph of all operators")
    g = gen(31)
    B, Hq, H, D, P, T, keep = 2, 8, 2, 128, 32, 150, 70
    cos, sin = (t.to(DEV) for t in rope_tables(D, 512, 10000.0))
    table, pages = table_for([T + 1] * B, P, g, spare=B * 3)
    used = set(table.flatten().tolist())
    new = torch.tensor([i for i in range(pages) if i not in used], dtype=torch.int32, device=DEV)[:B * 3].view(B, 3)
    pool = random_pool(pages, H, P, D, g)
    k, v, q = (randn(B, h, 1, D, g=g, dtype=torch.bfloat16) for h in (H, H, Hq))
    lens = torch.tensor([T, T - 40], dtype=torch.int32, device=DEV)
    lens_out = torch.empty_like(lens)

    def step():
        qh = nq.kv4_append(k, v, pool, table, q=q, cos=cos, sin=sin, pos_base=lens, row_base=lens, lens_out=lens_out)
        o, lse = nq.attention_decode_kv4(qh, pool, table, lens_out, max_len=T + 1, return_lse=True)
        w = nq.attention_key_weights(qh, pool, table, lens_out, lse, max_len=T + 1)
        kept = nq.select_keys(w, lens_out, keep=keep, recent=8, first=2)
        out = nq.kv_compact(pool, table, new, kept, weights=w)
        kr, vr = nq.kv4_gather(pool, new, S=keep)
        return o, lse, w, kept, out, kr, vr

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(3):
        for t in (k, v, q):
            t.copy_(randn(*t.shape, g=g))
        lens.copy_(torch.tensor([T - i, T - 50 - 3 * i]))
        graph.replay()
        got = [t.clone() for t in held]
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_side_stream_sees_its_own_inputs():
    say("another stream")
    g = gen(41)
    table, pages = table_for([3000], 64, g)
    pool = random_pool(pages, 2, 64, 128, g)
    lens = torch.tensor([3000], dtype=torch.int32, device=DEV)
    q = randn(1, 8, 128, g=g, dtype=torch.bfloat16)
    want = nq.attention_decode_kv4(q * 2, pool, table, lens, max_len=3000)
    big = torch.randn(4096, 4096, device=DEV)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        for _ in range(4):
            big = big @ big * 1e-2  # the stream is busy when the operators are queued
        q2 = q * 2
        o = nq.attention_decode_kv4(q2, pool, table, lens, max_len=3000)
    s.synchronize()
    assert torch.equal(o, want)


def test_plans_launch_again():
    say("plans")
    g = gen(51)
    table, pages = table_for([100], 32, g)
    pool = random_pool(pages, 1, 32, 64, g)
    lens = torch.tensor([100], dtype=torch.int32, device=DEV)
    q = randn(1, 4, 64, g=g, dtype=torch.bfloat16)
    call = nq.attention_decode_kv4(q, pool, table, lens, max_len=100, plan=True)
    first = call.launch().clone()
    q.mul_(-1)
    second = call.launch().clone()
    assert torch.equal(second, nq.attention_decode_kv4(q, pool, table, lens, max_len=100)) and not torch.equal(first, second)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("append", [False, True])
@pytest.mark.parametrize("Hq,max_len", [(4, 100), (8, 9000), (2, 33)])
def test_lse_of_paged_decodes_of_no_and_of_bad_lengths(Hq, max_len, append, dtype):
    """-inf without keys and NaN outside [0, max_len - append]: a merge and the key weights take
    -inf for "saw nothing", so a bad length must not look like one."""
    say(f"paged decode's lse {Hq}/2 max_len {max_len} append={append} {dtype}")
    g = gen(22)
    new = int(append)
    lens = [-1, 0, max_len - new, max_len - new + 1, 2 ** 30, 5]
    table, pages = table_for([max_len] * len(lens), 32, g)
    table = table.clamp(max=pages - 1)
    k, v = (randn(pages, 2, 32, 64, g=g, dtype=dtype) for _ in range(2))
    q = randn(len(lens), Hq, 64, g=g, dtype=dtype)
    kw = dict(max_len=max_len)
    if append:
        kw.update(k_new=randn(len(lens), 2, 64, g=g, dtype=dtype), v_new=randn(len(lens), 2, 64, g=g, dtype=dtype))
    o, lse = nq.attention_decode_paged(q, k, v, table, torch.tensor(lens, dtype=torch.int32, device=DEV), return_lse=True, **kw)
    bad = [0, 3, 4]
    assert torch.isnan(o[bad]).all() and torch.isnan(lse[bad]).all()
    good = [i for i in range(len(lens)) if i not in bad]
    assert torch.isfinite(o[good]).all()
    for b in good:
        n = lens[b] + new
        if n == 0:
            assert (o[b] == 0).all() and (lse[b] == -math.inf).all()
            continue
        _, want, _, spread = ref.attention(q[b], ref.rows_of(k, table[b], n).double(), ref.rows_of(v, table[b], n).double(), 1 / 8)
        # the bound of the lse test above (an appended row, not normed or rotated, is stored as it is)
        tol = spread * (2 * 64 + 8) * 2.0 ** -23 + (want.abs() + 1) * 2.0 ** -20 + (n + 64) * 2.0 ** -24
        assert ((lse[b].double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_operands_off_their_alignment(dtype):
    """Contiguous rows that start between 16-byte borders, and an axis of one with an odd stride."""
    say(f"misaligned operands {dtype}")
    g = gen(61)
    B, Hq, H, S, D, P, lens = 2, 8, 2, 3, 64, 32, [70, 33]

    def off(t):
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)
        out = buf[1:].view(t.shape)
        out.copy_(t)
        assert out.is_contiguous() and out.data_ptr() % 16
        return out

    table, pages = table_for([n + S for n in lens], P, g)
    pool = random_pool(pages, H, P, D, g)
    other = pool.clone()
    lens_t = torch.tensor(lens, dtype=torch.int32, device=DEV)
    k, v = (randn(B, H, S, D, g=g, dtype=dtype) for _ in range(2))
    q = randn(B, Hq, S, D, g=g, dtype=dtype)
    want = nq.kv4_append(k, v, pool, table, q=q, row_base=lens_t)
    assert torch.equal(nq.kv4_append(off(k), off(v), other, table, q=off(q), row_base=lens_t), want)
    assert torch.equal(pool, other)
    q1 = q[:, :, 0].contiguous()
    o, lse = nq.attention_decode_kv4(q1, pool, table, lens_t, max_len=70, return_lse=True)
    for t in (off(q1), q1.as_strided((B, Hq, 1, D), (Hq * D, D, 1, 1))):
        got, got_lse = nq.attention_decode_kv4(t, pool, table, lens_t, max_len=70, return_lse=True)
        assert torch.equal(got, o) and torch.equal(got_lse, lse)
    if dtype == torch.bfloat16:
        ls = torch.full((B, Hq, S), 4.0, device=DEV)
        w = nq.attention_key_weights(q, pool, table, lens_t, ls, max_len=70)
        assert torch.equal(nq.attention_key_weights(off(q), pool, table, lens_t, off(ls), max_len=70), w)
        one = nq.attention_key_weights(q1[:, :, None], pool, table, lens_t, lse, max_len=70)
        odd = q1.as_strided((B, Hq, 1, D), (Hq * D, D, 1, 1))
        assert torch.equal(nq.attention_key_weights(odd, pool, table, lens_t, lse, max_len=70), one)


def test_a_captured_loop_advances_its_lengths():
    """The step of the documentation: bounded by the rows that the table maps, its lengths advanced
    in the graph, over a page border; each replay as the eager step, and against the definition."""
    say("captured decode loop")
    g = gen(71)
    B, Hq, H, D, P, cols = 2, 8, 2, 64, 32, 4
    cos, sin = (t.to(DEV) for t in rope_tables(D, 512, 10000.0))
    table = torch.randperm(B * cols, generator=g, device=DEV).int().view(B, cols)
    pool = random_pool(B * cols, H, P, D, g)
    eager_pool = pool.clone()
    k, v, q = (randn(B, h, 1, D, g=g, dtype=torch.bfloat16) for h in (H, H, Hq))
    kw, qw = (1 + 0.1 * randn(D, g=g) for _ in range(2))
    start = [60, 91]

    def step(pool, lens, grown, w):
        qh = nq.kv4_append(k, v, pool, table, q=q, q_weight=qw, k_weight=kw, cos=cos, sin=sin, pos_base=lens,
                           row_base=lens, lens_out=grown)
        o, lse = nq.attention_decode_kv4(qh, pool, table, grown, max_len=cols * P, return_lse=True)
        nq.attention_key_weights(qh, pool, table, grown, lse, max_len=cols * P, weights=w)
        lens.add_(1)
        return qh, o, lse

    def state():
        lens = torch.tensor(start, dtype=torch.int32, device=DEV)
        return lens, torch.empty_like(lens), torch.zeros(B, H, cols * P, device=DEV)
    mine, theirs = state(), state()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(pool, *mine)
    torch.cuda.current_stream().wait_stream(side)
    pool.copy_(eager_pool)
    mine[0].copy_(torch.tensor(start))
    mine[2].zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(pool, *mine)
    for i in range(8):
        for t in (k, v, q):
            t.copy_(randn(*t.shape, g=g))
        graph.replay()
        got = [t.clone() for t in held]
        want = step(eager_pool, *theirs)
        torch.cuda.synchronize()
        for a, b in zip((*got, pool, *mine), (*want, eager_pool, *theirs)):
            assert torch.equal(a, b), i
        lens = [n + i + 1 for n in start]
        check_decode(got[1], got[2], got[0][:, :, 0], pool, table, lens, P, f"replay {i}")
    assert mine[0].tolist() == [n + 8 for n in start]
