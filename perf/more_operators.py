"""A KV cache held in 4 bits, and eviction by attention weight, as measurable cases.

A case is a dict of plain values.  ``kind`` selects the operators:

  rows     rows into 4-bit pages, and rows of those pages read back
  decode   a token's attention over 4-bit pages
  weights  the attention weight that each cached key got, summed over queries and heads
  evict    the keys worth keeping, and their rows moved to other pages

A 4-bit row holds blocks of 32 elements: codes of {0, 1/2, 1, 3/2, 2, 3, 4, 6} with a
sign, two a byte (the even element low), and a power of two per block, one byte with bias
127.  A page and head hold the K codes of all rows, the V codes, the K scales, the V scales.

Where ``own`` is true ``run`` calls the framework's operators, else the same formulas as
elementary tensor operations.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # the cache's share of one step of 64 users: each one's new row, at its own length
        dict(name="rows_step", kind="rows", B=64, Hkv=4, D=128, S=1, past=4000, ragged=True, P=64, dtype="bf16"),
        # a chunk of long prompts: its rows stored, and the whole history read back for its queries
        dict(name="rows_chunk", kind="rows", B=4, Hkv=8, D=128, S=2048, past=6144, ragged=False, P=64, dtype="bf16"),
        # prompts of no round size in an fp32 model
        dict(name="rows_odd_f32", kind="rows", B=3, Hkv=2, D=64, S=301, past=0, ragged=False, P=32, dtype="f32"),
        # one user's chat
        dict(name="decode_single", kind="decode", B=1, Hq=16, Hkv=8, D=128, T=512, ragged=False, P=64, dtype="bf16"),
        # a small batch at a common length
        dict(name="decode_batch", kind="decode", B=8, Hq=32, Hkv=8, D=128, T=4096, ragged=False, P=64, dtype="bf16"),
        # serving: many users at lengths up to a model's native context
        dict(name="decode_serving", kind="decode", B=64, Hq=64, Hkv=4, D=128, T=32768, ragged=True, P=64, dtype="bf16"),
        # an fp32 model, groups of no round size, a user without keys
        dict(name="decode_odd_f32", kind="decode", B=5, Hq=14, Hkv=2, D=64, T=3001, ragged=True, P=32, dtype="f32"),
        # the same serving step's weights, tracked for a later eviction
        dict(name="weights_step", kind="weights", B=64, Hq=64, Hkv=4, D=128, S=1, T=32768, ragged=True, P=64, cache="kv4"),
        # the last 64 tokens of long prompts say which of its keys matter
        dict(name="weights_window", kind="weights", B=4, Hq=32, Hkv=8, D=128, S=64, T=8192, ragged=False, P=64, cache="bf16"),
        # all of a shorter prompt's queries do
        dict(name="weights_prompt", kind="weights", B=2, Hq=16, Hkv=8, D=128, S=2048, T=2048, ragged=False, P=64, cache="bf16"),
        # a chat cut back to its budget
        dict(name="evict_small", kind="evict", B=2, Hkv=8, D=128, T=1500, keep=1000, recent=128, first=4, ragged=True, P=64,
             cache="kv4"),
        # long contexts cut to a quarter
        dict(name="evict_long", kind="evict", B=8, Hkv=8, D=128, T=32768, keep=8192, recent=256, first=4, ragged=False, P=64,
             cache="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rows", "decode", "weights", "evict"])
    D, P = rng.choice([32, 64, 128, 128]), rng.choice([32, 64, 96, 128])
    Hkv = rng.choice([1, 2, 4, 8])
    c = dict(kind=kind, Hkv=Hkv, D=D, P=P)
    if kind == "rows":
        S = 1 if rng.random() < 0.4 else _log_int(rng, 2, 4096)
        past = rng.choice([0, _log_int(rng, 1, 8192)])
        B = _log_int(rng, 1, min(64, max(1, (1 << 18) // ((S + past) * Hkv))))
        return dict(c, B=B, S=S, past=past, ragged=S == 1 and past > 0, dtype=rng.choice(["bf16", "bf16", "f32"]))
    if kind == "decode":
        T = _log_int(rng, 1, 65536)
        B = _log_int(rng, 1, min(64, max(1, (1 << 21) // (T * Hkv))))
        return dict(c, B=B, Hq=Hkv * rng.choice([1, 2, 4, 5, 8, 16]), T=T, ragged=rng.random() < 0.7,
                    dtype=rng.choice(["bf16", "bf16", "f32"]))
    if kind == "weights":
        S = rng.choice([1, 1, _log_int(rng, 2, 128), _log_int(rng, 64, 2048)])
        T = _log_int(rng, S, 32768)
        Hq = Hkv * rng.choice([1, 2, 4, 8])
        B = _log_int(rng, 1, min(32, max(1, (1 << 28) // (T * S * Hq * 4)), max(1, (1 << 21) // (T * Hkv))))
        return dict(c, B=B, Hq=Hq, S=S, T=T, ragged=rng.random() < 0.5, cache=rng.choice(["kv4", "bf16"]))
    T = _log_int(rng, 64, 65536)
    B = _log_int(rng, 1, min(32, max(1, (1 << 20) // (T * Hkv))))
    keep = max(8, int(T * rng.uniform(0.1, 0.9)))
    return dict(c, B=B, T=T, keep=keep, recent=keep // rng.choice([3, 8, 1000]), first=rng.choice([0, 1, 4]),
                ragged=rng.random() < 0.6, cache=rng.choice(["kv4", "bf16"]))


def _lens(case):
    """Cached rows of each sequence: of the case alone, since they decide its work."""
    B = case["B"]
    if case["kind"] == "rows":
        return [case["past"] - (17 * b % case["past"] if case["ragged"] else 0) for b in range(B)]
    T = case["T"]
    if not case["ragged"]:
        return [T] * B
    rng = random.Random(T * 1000 + B)
    lens = [rng.randint(max(case.get("S", 1), T // 32), T) for _ in range(B)]
    if case["kind"] == "decode" and 2 < B < 8:
        lens[1] = 0
    return lens


# ---------------------------------------------------------------- pages

def _quantise(x):
    """(codes, scale bytes) of fp32 rows (..., D)."""
    blocks = x.reshape(*x.shape[:-1], -1, 32)
    amax = blocks.abs().amax(-1)
    m, e = torch.frexp(amax)  # amax = m 2^e, m in [1/2, 1): the smallest scale with amax / scale <= 7
    e = torch.where(m <= 0.875, e - 3, e - 2)
    e = torch.where(amax > 0, e, -126).clamp(-126, 125)
    a = torch.ldexp(blocks.abs(), -e[..., None])
    code = torch.zeros_like(a, dtype=torch.uint8)
    # halfway goes to the even code
    for lo, at_least in ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (a >= lo) if at_least else (a > lo)
    code += (blocks < 0).to(torch.uint8) * 8
    return code.view(x.shape), (e + 127).to(torch.uint8)


def _values(codes, scales):
    """fp32 rows of codes (..., D) and scale bytes (..., D / 32)."""
    table = torch.tensor([*LEVELS, *(-v for v in LEVELS)], device=codes.device)
    v = table[codes.int()]
    s = torch.ldexp(torch.ones((), device=codes.device), scales.int() - 127)
    return (v.view(*v.shape[:-1], -1, 32) * s[..., None]).view(v.shape)


def _pack(codes):
    return codes[..., 0::2] | codes[..., 1::2] << 4


def _unpack(b):
    return torch.stack([b & 15, b >> 4], -1).flatten(-2)


def _page_parts(pages, D):
    """Views (K codes, V codes, K scales, V scales) of 4-bit pages (n, Hkv, P, 17 D / 16)."""
    n, H, P, _ = pages.shape
    flat = pages.view(n, H, -1)
    a, b = P * D // 2, P * D // 32
    return (flat[..., :a].view(n, H, P, D // 2), flat[..., a:2 * a].view(n, H, P, D // 2),
            flat[..., 2 * a:2 * a + b].view(n, H, P, D // 32), flat[..., 2 * a + b:].view(n, H, P, D // 32))


def _read_pages(pool, page_ids, D):
    """fp32 K and V (Hkv, rows, D) of a sequence's 4-bit pages."""
    kc, vc, ks, vs = _page_parts(pool[page_ids], D)
    return [_values(_unpack(c), s).transpose(0, 1).reshape(pool.shape[1], -1, D) for c, s in ((kc, ks), (vc, vs))]


def _rows(shape, g):
    """Normalised and rotated keys, or values: some dimensions far larger than others."""
    x = torch.randn(shape, generator=g, device=DEV)
    return x * (1 + 3 * (torch.arange(shape[-1], device=DEV) % 29 == 3))


def _tables(case, lens, g, extra=0):
    """(block table, pages) with pages in no order; ``extra`` further pages behind them."""
    P = case["P"]
    need = [-(-n // P) for n in lens]
    ids = torch.randperm(sum(need), generator=g, device=DEV).int()
    table = torch.zeros(len(lens), max(max(need), 1), dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    return table, max(at, 1) + extra


def _fill_kv4(pool, g, D):
    for i in range(0, pool.shape[0], 1024):
        part = pool[i:i + 1024]
        for c, s in zip(_page_parts(part, D)[:2], _page_parts(part, D)[2:]):
            codes, scales = _quantise(_rows((*c.shape[:3], D), g))
            c.copy_(_pack(codes))
            s.copy_(scales)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    B, Hkv, D, P, kind = (case[k] for k in ("B", "Hkv", "D", "P", "kind"))
    lens = _lens(case)
    s = dict(case=case, host_lens=lens, lens=torch.tensor(lens, dtype=torch.int32, device=DEV))
    if kind == "rows":
        s["table"], pages = _tables(case, [n + case["S"] for n in lens], g)
        s["pool"] = torch.zeros(pages, Hkv, P, 17 * D // 16, dtype=torch.uint8, device=DEV)
        if case["past"] and not case["ragged"]:
            _fill_kv4(s["pool"], g, D)
        for name in ("k", "v"):  # as projections leave them
            s[name] = _rows((B, case["S"], Hkv, D), g).to(DTYPES[case["dtype"]]).transpose(1, 2)
        return s
    if kind == "evict":
        new_pages = B * -(-case["keep"] // P)
        s["table"], pages = _tables(case, lens, g, extra=new_pages)
        first_new = pages - new_pages
        s["new_table"] = torch.arange(first_new, pages, dtype=torch.int32, device=DEV).view(B, -1)
        s["first_new"] = first_new
        # few keys have most of the weight, the latest ones have had little time to get any
        w = torch.exp(2 * torch.randn(B, Hkv, case["T"], generator=g, device=DEV))
        w *= torch.rand(B, Hkv, case["T"], generator=g, device=DEV) > 0.1
        s["weights"] = w
    else:
        s["table"], pages = _tables(case, lens, g)
    if case.get("cache", "kv4") == "kv4":
        s["pool"] = torch.zeros(pages, Hkv, P, 17 * D // 16, dtype=torch.uint8, device=DEV)
        _fill_kv4(s["pool"][:s.get("first_new", pages)], g, D)
    else:
        s["k_pool"], s["v_pool"] = (torch.zeros(pages, Hkv, P, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        for pool in (s["k_pool"], s["v_pool"])[:2 if kind == "evict" else 1]:
            for i in range(0, s.get("first_new", pages), 1024):
                part = pool[i:min(i + 1024, s.get("first_new", pages))]
                part.copy_(_rows(part.shape, g))
    if kind == "decode":
        s["q"] = _rows((B, case["Hq"], D), g).to(DTYPES[case["dtype"]])
    if kind == "weights":
        s["q"] = _rows((B, case["S"], case["Hq"], D), g).bfloat16().transpose(1, 2)
        s["lse"] = torch.stack([_scores(s, b, torch.float32).logsumexp(-1).view(case["Hq"], -1) for b in range(B)])
    return s


# ---------------------------------------------------------------- the framework's operators

def _own(s):
    import nano_qwen_amd as nq
    c = s["case"]
    if c["kind"] == "rows":
        if c["ragged"]:
            nq.kv4_append(s["k"], s["v"], s["pool"], s["table"], row_base=s["lens"])
            return list(nq.kv4_gather(s["pool"], s["table"], S=c["S"], row_base=s["lens"], dtype=DTYPES[c["dtype"]]))
        nq.kv4_append(s["k"], s["v"], s["pool"], s["table"], row_offset=c["past"])
        return list(nq.kv4_gather(s["pool"], s["table"], S=c["past"] + c["S"], dtype=DTYPES[c["dtype"]]))
    if c["kind"] == "decode":
        return [nq.attention_decode_kv4(s["q"], s["pool"], s["table"], s["lens"], max_len=max(s["host_lens"]))]
    if c["kind"] == "weights":
        pool = s["pool"] if c["cache"] == "kv4" else s["k_pool"]
        longest = max(s["host_lens"])
        w = None if longest == c["T"] else torch.zeros(c["B"], c["Hkv"], c["T"], device=DEV)
        return [nq.attention_key_weights(s["q"], pool, s["table"], s["lens"], s["lse"], max_len=longest, weights=w)]
    kept = nq.select_keys(s["weights"], s["lens"], keep=c["keep"], recent=c["recent"], first=c["first"])
    pools = s["pool"] if c["cache"] == "kv4" else (s["k_pool"], s["v_pool"])
    w = nq.kv_compact(pools, s["table"], s["new_table"], kept, weights=s["weights"])
    if c["cache"] == "kv4":
        return [kept, w, *nq.kv4_gather(s["pool"], s["new_table"], S=c["keep"])]
    return [kept, w, s["k_pool"][s["first_new"]:], s["v_pool"][s["first_new"]:]]


# ---------------------------------------------------------------- the plain forms

def _scores(s, b, dtype):
    """(Hkv, G S, T) scaled scores of sequence b, -inf where a query does not see a key."""
    c = s["case"]
    Hkv, D, n, P = c["Hkv"], c["D"], s["host_lens"][b], c["P"]
    ids = s["table"][b, :-(-n // P)].long()
    if c["cache"] == "kv4":
        k = _read_pages(s["pool"], ids, D)[0][:, :n].to(dtype)
    else:
        k = s["k_pool"][ids].transpose(0, 1).reshape(Hkv, -1, D)[:, :n].to(dtype)
    S = c["S"]
    q = s["q"][b].to(dtype).reshape(Hkv, -1, D)
    x = torch.matmul(q, k.transpose(1, 2).contiguous()) / math.sqrt(D)
    if S > 1:
        t, i = torch.arange(n, device=DEV), torch.arange(S, device=DEV)
        hidden = t[None, :] > i[:, None] + (n - S)
        x.view(Hkv, -1, S, n).masked_fill_(hidden, -math.inf)
    return x


def _plain(s):
    c = s["case"]
    B, Hkv, D, P, lens = c["B"], c["Hkv"], c["D"], c["P"], s["host_lens"]
    if c["kind"] == "rows":
        out, dtype = [], DTYPES[c["dtype"]]
        for i, x in enumerate((s["k"], s["v"])):
            new = _values(*_quantise(x.float()))
            if c["past"] and not c["ragged"]:
                old = [_read_pages(s["pool"], s["table"][b].long(), D)[i][:, :c["past"]] for b in range(B)]
                new = torch.cat([torch.stack(old), new], 2)
            out.append(new.to(dtype))
        return out
    if c["kind"] == "decode":
        out = torch.zeros_like(s["q"])
        for b in range(B):
            n = lens[b]
            if n == 0:
                continue
            k, v = (x[:, :n] for x in _read_pages(s["pool"], s["table"][b, :-(-n // P)].long(), D))
            q = s["q"][b].float().view(Hkv, -1, D).transpose(1, 2).contiguous()
            x = torch.matmul(k, q) / math.sqrt(D)  # (Hkv, T, G)
            p = torch.exp(x - x.amax(1, keepdim=True))
            o = torch.matmul(p.transpose(1, 2).contiguous(), v) / p.sum(1)[..., None]
            out[b] = o.view(-1, D).to(out.dtype)
        return [out]
    if c["kind"] == "weights":
        w = torch.zeros(B, Hkv, c["T"], device=DEV)
        for b in range(B):
            p = torch.exp(_scores(s, b, torch.float32) - s["lse"][b].view(Hkv, -1, 1))
            w[b, :, :lens[b]] = p.sum(1)
        return [w]
    t, n, keep = torch.arange(c["T"], device=DEV), s["lens"][:, None, None], c["keep"]
    rank = torch.where((t < c["first"]) | (t >= n - c["recent"]), math.inf, s["weights"])
    rank = torch.where(t < n, rank, -math.inf)
    kept = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep].sort(-1).values
    kept = torch.where(kept < n, kept, c["T"]).sort(-1).values
    real = kept < c["T"]
    at = torch.where(real, kept, 0)
    w = torch.zeros_like(s["weights"])
    w[..., :keep] = torch.where(real, s["weights"].gather(-1, at), 0.0)
    pages = s["table"].long()[:, None].gather(-1, (at // P).view(B, 1, -1)).view(at.shape)
    heads = torch.arange(Hkv, device=DEV)[:, None]
    new_pages = s["new_table"].long()[:, None].repeat_interleave(P, -1)[..., :keep].expand(-1, Hkv, -1)
    to = new_pages, heads.expand_as(kept), t[:keep].expand_as(kept) % P
    kept = torch.where(real, kept, -1).int()
    if c["cache"] == "kv4":
        kc, vc, ks, vs = _page_parts(s["pool"], D)
        return [kept, w, *(torch.where(real[..., None], _values(_unpack(x[pages, heads, at % P]), e[pages, heads, at % P]),
                                       0.0).bfloat16() for x, e in ((kc, ks), (vc, vs)))]
    out = [kept, w]
    for pool in (s["k_pool"], s["v_pool"]):
        pool[to] = torch.where(real[..., None], pool[pages, heads, at % P], pool[to])
        out.append(pool[s["first_new"]:])
    return out


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _plain(state)


def work(case):
    B, Hkv, D = case["B"], case["Hkv"], case["D"]
    lens, row4 = _lens(case), 17 * D // 16
    total = Hkv * sum(lens)
    if case["kind"] == "rows":
        e = 2 if case["dtype"] == "bf16" else 4
        new = B * Hkv * case["S"]
        read = new if case["ragged"] else new + total
        return dict(bytes=new * (2 * D * e + row4) + read * (row4 + 2 * D * e), flops=8 * D * (new + read))
    if case["kind"] == "decode":
        e = 2 if case["dtype"] == "bf16" else 4
        return dict(bytes=total * row4 + 2 * B * case["Hq"] * D * e, flops=4 * D * case["Hq"] * sum(lens))
    if case["kind"] == "weights":
        S, Hq = case["S"], case["Hq"]
        pairs = sum(S * n - S * (S - 1) // 2 for n in lens)
        k = row4 // 2 if case["cache"] == "kv4" else 2 * D
        return dict(bytes=total * k + B * S * Hq * (2 * D + 4) + 4 * B * Hkv * case["T"], flops=2 * D * Hq * pairs)
    row = row4 if case["cache"] == "kv4" else 4 * D
    kept = Hkv * sum(min(n, case["keep"]) for n in lens)
    back = B * Hkv * case["keep"] * (row4 + 4 * D) if case["cache"] == "kv4" else 0
    return dict(bytes=4 * total + kept * 2 * row + 4 * B * Hkv * (case["keep"] + case["T"]) + back, flops=8 * total)


# ---------------------------------------------------------------- the definitions in 64 bits

def _exact_stored(x):
    """What rows stand for once stored: the nearest multiple of the block's scale that a code has."""
    blocks = x.double().reshape(*x.shape[:-1], -1, 32)
    top = blocks.abs().amax(-1, keepdim=True)
    scale = torch.full_like(top, 2.0 ** -126)
    while bool((grow := (top > 7 * scale) & (scale < 2.0 ** 125)).any()):
        scale = torch.where(grow, 2 * scale, scale)
    y = blocks.abs() / scale
    best, gap = torch.zeros_like(y), y.clone()
    for code, level in enumerate(LEVELS[1:], 1):
        d = (y - level).abs()
        nearer = d < gap if code % 2 else d <= gap
        best, gap = torch.where(nearer, level, best), torch.where(nearer, d, gap)
    return (torch.sign(blocks) * best * scale).view(x.shape)


def _exact_read(pages, which):
    """Rows (Hkv, n P, D) of 4-bit pages in 64 bits: which = 0 for K, 1 for V."""
    n, H, P, row = pages.shape
    D = row * 16 // 17
    raw = pages.reshape(n, H, -1).long()
    codes = raw[..., which * P * D // 2:(which + 1) * P * D // 2].reshape(n, H, P, D // 2, 1)
    codes = (codes >> torch.tensor([0, 4], device=raw.device)) & 15
    at = P * D + which * P * D // 32
    e = raw[..., at:at + P * D // 32].reshape(n, H, P, D // 32, 1).double() - 127
    magnitude, exponent = codes & 1, (codes >> 1) & 3
    v = torch.where(exponent > 0, (1 + magnitude / 2.0) * 2.0 ** (exponent.double() - 1), magnitude / 2.0)
    v = v.double() * (1 - 2 * (codes >> 3))
    return (v.view(n, H, P, D // 32, 32) * 2.0 ** e).view(n, H, P, D).transpose(0, 1).reshape(H, n * P, D)


def exact(case, seed):
    s = prepare(case, seed)
    B, Hkv, D, P, kind, lens = case["B"], case["Hkv"], case["D"], case["P"], case["kind"], s["host_lens"]

    def pages(b, n):
        return s["pool"][s["table"][b, :-(-n // P)].long()]

    if kind == "rows":
        out = []
        for i, x in enumerate((s["k"], s["v"])):
            new = _exact_stored(x)
            if case["past"] and not case["ragged"]:
                new = torch.cat([torch.stack([_exact_read(pages(b, case["past"]), i)[:, :case["past"]] for b in range(B)]),
                                 new], 2)
            out.append(new)
        return out
    if kind == "decode":
        out = torch.zeros(B, case["Hq"], D, dtype=torch.float64, device=DEV)
        for b, n in enumerate(lens):
            if n:
                k, v = (_exact_read(pages(b, n), i)[:, :n] for i in (0, 1))
                z = torch.matmul(s["q"][b].double().view(Hkv, -1, D), k.transpose(1, 2).contiguous()) * D ** -0.5
                out[b] = torch.matmul(torch.softmax(z, -1), v).view(-1, D)
        return [out]
    if kind == "weights":
        S, Hq = case["S"], case["Hq"]
        w = torch.zeros(B, Hkv, case["T"], dtype=torch.float64, device=DEV)
        for b, n in enumerate(lens):
            if case["cache"] == "kv4":
                k = _exact_read(pages(b, n), 0)[:, :n]
            else:
                k = s["k_pool"][s["table"][b, :-(-n // P)].long()].double().transpose(0, 1).reshape(Hkv, -1, D)[:, :n]
            sees = torch.ones(S, n, dtype=torch.bool, device=DEV).tril(n - S)
            for h in range(Hq):
                g = h * Hkv // Hq
                z = s["q"][b, h].double() @ k[g].t().contiguous() * D ** -0.5 - s["lse"][b, h].double()[:, None]
                w[b, g, :n] += torch.where(sees, torch.exp(z), 0.0).sum(0)
        return [w]
    T, keep = case["T"], case["keep"]
    kept = torch.full((B, Hkv, keep), -1, dtype=torch.int32, device=DEV)
    w = torch.zeros(B, Hkv, T, dtype=torch.float64, device=DEV)
    if case["cache"] == "kv4":
        out = [torch.zeros(B, Hkv, keep, D, dtype=torch.float64, device=DEV) for _ in range(2)]
    else:
        out = [s[p][s["first_new"]:].double() for p in ("k_pool", "v_pool")]
    for b, n in enumerate(lens):
        if case["cache"] == "kv4":
            rows = [_exact_read(pages(b, n), i) for i in (0, 1)]
        else:
            rows = [s[p][s["table"][b, :-(-n // P)].long()].double().transpose(0, 1).reshape(Hkv, -1, D)
                    for p in ("k_pool", "v_pool")]
        for h in range(Hkv):
            idx = torch.arange(n, device=DEV)
            if n > keep:
                free = idx[case["first"]:n - case["recent"]]
                room = keep - case["first"] - case["recent"]
                v = s["weights"][b, h][free].double()
                limit = torch.sort(v).values[len(v) - room] if room else math.inf
                above = v > limit
                ties = torch.nonzero(v == limit)[:, 0][:room - int(above.sum())]
                above[ties] = True
                idx = torch.cat([idx[:case["first"]], free[above], idx[n - case["recent"]:]])
            m = len(idx)
            kept[b, h, :m] = idx.int()
            w[b, h, :m] = s["weights"][b, h][idx].double()
            for o, r in zip(out, rows):
                if case["cache"] == "kv4":
                    o[b, h, :m] = r[h, idx]
                else:
                    j = torch.arange(m, device=DEV)
                    o[b * -(-keep // P) + j // P, h, j % P] = r[h, idx]
    return [kept, w, *out]
