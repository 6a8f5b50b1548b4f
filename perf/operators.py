"""Cases and plain forms of the 4-bit paged KV-cache operators.

Four calls on one attention layer's cache are measured, as a serving loop makes
them: append (per-head q / k RMSNorm, partial rotation, 4-bit quantisation and
the write into the pages), attention over the cached pages (one token per
sequence, a few, or a prefill chunk; optionally with the log-sum-exp and the
weight every cached key received), eviction of the keys with the least
accumulated weight, and the read of cached tokens back as the values they stand
for (the append and eviction cases return the cache through it).

A page holds 16 tokens. Of each (page, KV head) it keeps one block of 18 x D
bytes: K nibbles (8 D), V nibbles (8 D), then K and V scale / bias pairs (bf16)
of every token's groups of 64 values (D each). A value is scale * n + bias with
n in 0..15. `own` chooses between these plain forms and the framework's calls.
"""
import math

import numpy as np
import torch

own = False

PAGE = 16
GROUP = 64
KINDS = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SMALL = dict(q_heads=4, kv_heads=1, head_dim=64, rope=16)      # the tiny hybrid decoder of the tests
LARGE = dict(q_heads=16, kv_heads=2, head_dim=256, rope=64)    # the benchmark's attention layers


def listed():
    return [
        # eight decoding sequences of the tiny decoder: the smallest call, all latency
        dict(name="append_8_small", op="append", tokens=8, kind="f16", context=256, fused=False, **SMALL),
        # one decode step of 64 sequences at the benchmark's widths
        dict(name="append_64", op="append", tokens=64, kind="bf16", context=32768, fused=True, **LARGE),
        # a chunked-prefill step's rows (2048 prompt tokens and 120 decode tokens) read from fp32 projection rows
        dict(name="append_2168", op="append", tokens=2168, kind="f32", context=16384, fused=True, **LARGE),
        # eight short sequences of the tiny decoder
        dict(name="attention_8_small", op="attention", seqs=8, tokens=1, low=1, high=256, kind="f16", gate=False,
             ragged=False, stats=False, **SMALL),
        # the benchmark's decode batch: 64 sequences, contexts log-uniform in [128, 32768], gated output
        dict(name="attention_64", op="attention", seqs=64, tokens=1, low=128, high=32768, kind="bf16", gate=True,
             ragged=False, stats=False, **LARGE),
        # generic widths, an odd number of sequences and odd lengths
        dict(name="attention_33_d128", op="attention", seqs=33, tokens=1, low=17, high=5003, kind="f16", gate=False,
             ragged=False, stats=False, q_heads=20, kv_heads=4, head_dim=128, rope=128),
        # speculative verification: up to four tokens fed per sequence
        dict(name="attention_verify_128", op="attention", seqs=128, tokens=4, low=128, high=8192, kind="bf16", gate=True,
             ragged=True, stats=False, **LARGE),
        # one chunk of a long prompt: 2048 tokens over 16384 cached keys
        dict(name="attention_chunk_2048", op="attention", seqs=1, tokens=2048, low=16384, high=16384, kind="bf16",
             gate=True, ragged=False, stats=False, **LARGE),
        # decode that also accumulates what every cached key received (a cache that will be evicted from)
        dict(name="attention_weights_32", op="attention", seqs=32, tokens=1, low=256, high=16384, kind="bf16", gate=False,
             ragged=False, stats=True, **LARGE),
        # eviction on the tiny decoder
        dict(name="evict_8_small", op="evict", seqs=8, low=40, high=500, keep=100, recent=16, **SMALL),
        # long contexts cut to 4096 keys per KV head
        dict(name="evict_32", op="evict", seqs=32, low=2048, high=32768, keep=4096, recent=256, **LARGE),
    ]


def draw(rng):
    def log(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    heads = rng.choice([SMALL, LARGE, dict(q_heads=20, kv_heads=4, head_dim=128, rope=128),
                        dict(q_heads=6, kv_heads=6, head_dim=64, rope=32), dict(q_heads=32, kv_heads=2, head_dim=128, rope=0)])
    op = rng.choice(["append", "attention", "attention", "attention", "evict"])
    if op == "append":
        return dict(op=op, tokens=log(1, 2168), kind=rng.choice(list(KINDS)), context=log(64, 32768),
                    fused=rng.random() < 0.5, **heads)
    if op == "evict":
        high = log(100, 32768)
        keep = log(8, min(4096, high))
        return dict(op=op, seqs=log(1, 32), low=log(max(1, high // 16), high), high=high, keep=keep,
                    recent=rng.randrange(keep + 1), **heads)
    tokens = rng.choice([1, 1, rng.randrange(2, 9), log(9, 1024)])
    most = 8192 if heads["head_dim"] == 256 else 4096
    high = max(tokens, log(16, most))
    seqs = max(1, min(log(1, 96), 2 ** 21 // (high * max(1, tokens // 4))))
    return dict(op=op, seqs=seqs, tokens=tokens, low=log(max(1, high // 64), high), high=high,
                kind=rng.choice(["f16", "bf16"]), gate=rng.random() < 0.5, ragged=rng.random() < 0.5,
                stats=rng.random() < 0.3, **heads)


# ------------------------------------------------------------------ the page layout

_tables = {}


def _places(head_dim, device):
    """Where the values of a (page, KV head) block are: for K and V the byte [token, dim] and shift [dim] of a
    nibble, for each of a token's bytes (in byte order) the dims of its low and high nibble, and the
    scale / bias places [token, group]."""
    at = _tables.get((head_dim, device))
    if at is not None:
        return at
    D, words = head_dim, head_dim // 32  # K words of one lane
    tok, dim = torch.arange(PAGE)[:, None], torch.arange(D)[None, :]
    # K: dim = 64 group + 32 half + 8 lane + e in word 2 group + half of `lane`; e in nibble e / 2 + 4 (e % 2)
    word, lane, e = 2 * (dim // 64) + dim % 64 // 32, dim % 32 // 8, dim % 8
    chunk = min(words, 4)
    nib = e // 2 + 4 * (e % 2)
    k_byte = ((word // chunk * PAGE + tok) * 4 + lane) * chunk * 4 + word % chunk * 4 + nib // 2
    k_shift = (nib % 2 * 4).expand(PAGE, D)[0]
    # V: dim = 64 group + 8 lane + e in word `group` of `lane`; e in nibble e; even tokens before odd ones
    group, lane, e = dim // 64, dim % 64 // 8, dim % 8
    per, order = 512 // D, tok % 2 * 8 + tok // 2
    v_byte = 8 * D + (lane // per * PAGE + order) * 32 + lane % per * (D // 16) + group * 4 + e // 2
    v_shift = (e % 2 * 4).expand(PAGE, D)[0]

    def bytes_of(byte, shift):
        first = byte[0]
        order = torch.argsort(first * 2 + shift // 4)
        return byte[:, order[0::2]], order[0::2], order[1::2]  # [token, D / 2], low dims, high dims

    k_bytes, k_low, k_high = bytes_of(k_byte, k_shift)
    v_bytes, v_low, v_high = bytes_of(v_byte, v_shift)
    meta = torch.arange(PAGE)[:, None] * (D // GROUP) + torch.arange(D // GROUP)[None, :]
    at = dict(k_byte=k_byte, k_shift=k_shift, v_byte=v_byte, v_shift=v_shift, k_bytes=k_bytes, k_low=k_low,
              k_high=k_high, v_bytes=v_bytes, v_low=v_low, v_high=v_high, k_meta=16 * D + 4 * meta,
              v_meta=17 * D + 4 * meta)
    at = {k: v.to(device) for k, v in at.items()}
    _tables[head_dim, device] = at
    return at


def _values(block, head_dim):
    """K and V of blocks [..., 18 D] as fp32 [..., token, D]."""
    p, out = _places(head_dim, block.device), []
    for byte, shift, meta in (("k_byte", "k_shift", "k_meta"), ("v_byte", "v_shift", "v_meta")):
        n = (block[..., p[byte]] >> p[shift].to(torch.uint8)) & 15
        pair = block[..., 16 * head_dim:] if byte[0] == "k" else block[..., 17 * head_dim:]
        pair = pair[..., :head_dim].contiguous().view(torch.bfloat16).unflatten(-1, (PAGE, head_dim // GROUP, 2)).float()
        scale, bias = pair[..., 0, None], pair[..., 1, None]
        out.append((scale * n.unflatten(-1, (-1, GROUP)).float() + bias).flatten(-2))
    return out


def _quantise(x):
    """(nibbles [..., D] uint8, pairs [..., D / 64, 2] bf16) of values in 64 bits."""
    g = x.unflatten(-1, (-1, GROUP))
    low, high = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    scale = ((high - low) / 15).float().bfloat16()
    bias = low.float().bfloat16()
    s = scale.double()
    n = torch.where(s > 0, ((g - bias.double()) / torch.where(s > 0, s, 1.0)).round().clamp(0, 15), 0.0)
    return n.to(torch.uint8).flatten(-2), torch.cat([scale, bias], -1)


def _store(pool, head_dim, slots, k, v):
    """Writes tokens [T, KV head, D] (64 bits) at their slots."""
    p, page, at = _places(head_dim, pool.device), slots // PAGE, slots % PAGE
    heads = torch.arange(k.shape[1], device=pool.device)[None, :, None]
    for x, name in ((k, "k"), (v, "v")):
        n, pair = _quantise(x)
        packed = n[..., p[name + "_low"]] | (n[..., p[name + "_high"]] << 4)
        pool[page[:, None, None], heads, p[name + "_bytes"][at][:, None, :]] = packed
        meta = (p[name + "_meta"][at][:, None, :, None] + torch.arange(4, device=pool.device)).flatten(-2)
        pool[page[:, None, None], heads, meta] = pair.contiguous().view(torch.uint8).flatten(-2)


# ------------------------------------------------------------------ inputs

def _lengths(case):
    n = case["seqs"]
    low, high = math.log(case["low"]), math.log(case["high"])
    return [max(1, round(math.exp(low + (high - low) * (i + 0.5) / n))) for i in range(n)]


def _counts(case, lens):
    n = case["tokens"]
    return [min(m, max(1, n * (i % 4 + 1) // 4) if case["ragged"] else n) for i, m in enumerate(lens)]  # a token is cached before it is asked for


def _filled_pool(case, pages, gen):
    """Pages of quantised values: keys with a few strong channels, as after a rotation, and values of varied size."""
    D, H, dev = case["head_dim"], case["kv_heads"], "cuda"
    p = _places(D, torch.device("cuda", torch.cuda.current_device()))
    pool = torch.empty(pages, H, 18 * D, dtype=torch.uint8, device=dev)
    strong = 1 + 3 * (torch.rand(H, 1, D, generator=gen, device=dev) < 0.03).float()
    for a in range(0, pages, 4096):
        b = min(pages, a + 4096)
        k = torch.randn(b - a, H, PAGE, D, generator=gen, device=dev) * strong
        v = torch.randn(b - a, H, PAGE, D, generator=gen, device=dev)
        v *= 0.25 + torch.rand(b - a, H, PAGE, 1, generator=gen, device=dev)
        for x, name in ((k, "k"), (v, "v")):
            n, pair = _quantise(x)
            block = pool[a:b]
            packed = n[..., p[name + "_low"]] | (n[..., p[name + "_high"]] << 4)
            block[..., p[name + "_bytes"].flatten()] = packed.flatten(-2)
            at = 16 * D if name == "k" else 17 * D
            block[..., at:at + D] = pair.contiguous().view(torch.uint8).flatten(2)
    return pool


def _table(lens, gen, first=0):
    """Block tables [seqs, pages of the longest] over shuffled pages, and the number of pages."""
    need = [-(-n // PAGE) for n in lens]
    ids = torch.randperm(sum(need), generator=gen, device="cuda").to(torch.int32) + first
    table = torch.zeros(len(lens), max(need), dtype=torch.int32, device="cuda")
    cols = torch.arange(max(need), device="cuda")[None, :]
    table[cols < torch.tensor(need, device="cuda")[:, None]] = ids
    return table, sum(need)


def _package():
    import importlib
    return importlib.import_module("rust-ts-tokio-inference-engine_b200")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    Hq, Hkv, D = case["q_heads"], case["kv_heads"], case["head_dim"]
    s = dict(case=case)

    def ints(x, kind=torch.int32):
        return torch.tensor(x, dtype=kind, device="cuda")

    if case["op"] == "append":
        T, kind = case["tokens"], KINDS[case["kind"]]
        pages = -(-T // PAGE) * 2 + 1
        s["pool"] = torch.zeros(pages, Hkv, 18 * D, dtype=torch.uint8, device="cuda")
        s["slots"] = torch.randperm(pages * PAGE, generator=gen, device="cuda")[:T].contiguous()
        s["positions"] = torch.randint(0, case["context"], (T,), generator=gen, device="cuda", dtype=torch.int32)
        if case["fused"]:  # rows of the input projection: [query, gate] per query head, keys, values
            row = torch.randn(T, (2 * Hq + 2 * Hkv) * D, generator=gen, device="cuda").to(kind)
            s["q"] = row[:, :2 * Hq * D].view(T, Hq, 2, D)[:, :, 0]
            s["k"] = row[:, 2 * Hq * D:(2 * Hq + Hkv) * D].view(T, Hkv, D)
            s["v"] = row[:, (2 * Hq + Hkv) * D:].view(T, Hkv, D)
        else:
            for name, heads in (("q", Hq), ("k", Hkv), ("v", Hkv)):
                s[name] = torch.randn(T, heads, D, generator=gen, device="cuda").to(kind)
        s["q_norm"] = 1 + 0.1 * torch.randn(D, generator=gen, device="cuda")
        s["k_norm"] = 1 + 0.1 * torch.randn(D, generator=gen, device="cuda")
    elif case["op"] == "attention":
        lens, kind = _lengths(case), KINDS[case["kind"]]
        counts = _counts(case, lens)
        order = torch.randperm(len(lens), generator=gen, device="cuda").tolist()
        lens, counts = [lens[i] for i in order], [counts[i] for i in order]
        T = sum(counts)
        s["table"], pages = _table(lens, gen)
        s["pool"] = _filled_pool(case, pages, gen)
        s["lens"] = ints(lens)
        s["cu"] = ints([sum(counts[:i]) for i in range(len(counts) + 1)])
        s["q"] = torch.randn(T, Hq, D, generator=gen, device="cuda").to(kind)
        s["gate"] = torch.randn(T, Hq, D, generator=gen, device="cuda") if case["gate"] else None
        s["weights"] = None
        if case["stats"]:
            width = s["table"].shape[1] * PAGE
            s["weights"] = torch.rand(len(lens), Hkv, width, generator=gen, device="cuda") ** 8
            s["new_weights"] = s["weights"].clone()  # columns behind a sequence's length stay as they are
    else:
        lens = _lengths(case)
        lens = [lens[i] for i in torch.randperm(len(lens), generator=gen, device="cuda").tolist()]
        s["table"], pages = _table(lens, gen)
        kept = [min(n, case["keep"]) for n in lens]
        s["new_table"], more = _table(kept, gen, pages)
        s["pool"] = torch.zeros(pages + more, Hkv, 18 * D, dtype=torch.uint8, device="cuda")
        s["pool"][:pages] = _filled_pool(case, pages, gen)
        s["lens"] = ints(lens)
        s["weights"] = torch.rand(len(lens), Hkv, s["table"].shape[1] * PAGE, generator=gen, device="cuda") ** 8
        # the slots that the kept keys are read back from, sequence by sequence
        at = torch.arange(max(kept), device="cuda")[None, :]
        slots = s["new_table"].long().repeat_interleave(PAGE, 1)[:, :max(kept)] * PAGE + at % PAGE
        s["slots"] = slots[at < ints(kept)[:, None]].contiguous()
    if own:
        K = _package()
        s["cache"] = K.Kv4Cache(s["pool"], Hq, Hkv, D)
        if case["op"] == "attention":
            s["workspace"] = torch.empty(s["cache"].workspace_bytes(len(counts), T), dtype=torch.uint8, device="cuda")
    return s


# ------------------------------------------------------------------ the operators

EPS, THETA = 1e-6, 1e7


def _rotated(x, positions, rope):
    """Halves (j, j + rope / 2) of the first `rope` dims turned by position * theta^(-2 j / rope); angles in 64 bits."""
    if not rope:
        return x
    j = torch.arange(rope // 2, device=x.device, dtype=torch.float64)
    angle = positions.double()[:, None, None] * THETA ** (-2.0 * j / rope)
    c, n = angle.cos(), angle.sin()
    a, b = x[..., :rope // 2], x[..., rope // 2:rope]
    return torch.cat([(a * c - b * n).to(x.dtype), (a * n + b * c).to(x.dtype), x[..., rope:]], -1)


def _normed(x, w):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.to(x.dtype)


def _cached(pool, head_dim, slots):
    """K and V [T, KV head, D] of cached tokens."""
    k, v = _values(pool[slots // PAGE], head_dim)
    at = (slots % PAGE)[:, None, None, None].expand(-1, k.shape[1], 1, head_dim)
    return k.gather(2, at)[:, :, 0], v.gather(2, at)[:, :, 0]


def _append(s):
    c = s["case"]
    if own:
        T, dev = c["tokens"], s["q"].device
        q = torch.empty(T, c["q_heads"], c["head_dim"], dtype=torch.bfloat16 if c["kind"] == "f32" else s["q"].dtype, device=dev)
        k = torch.empty(T, c["kv_heads"], c["head_dim"], dtype=torch.float32, device=dev)
        v = torch.empty_like(k)
        s["cache"].append(s["q"], s["k"], s["v"], s["positions"], s["slots"], q, q_norm=s["q_norm"], k_norm=s["k_norm"],
                          epsilon=EPS, theta=THETA, rope_dims=c["rope"])
        s["cache"].read(s["slots"], k, v)
        return dict(q=q, k=k, v=v)
    q = _rotated(_normed(s["q"].float(), s["q_norm"]), s["positions"], c["rope"])
    # a key one rounding away from a border between two nibbles would differ by a whole step: 64 bits
    k = _rotated(_normed(s["k"].double(), s["k_norm"]), s["positions"], c["rope"])
    _store(s["pool"], c["head_dim"], s["slots"], k, s["v"].double())
    k, v = _cached(s["pool"], c["head_dim"], s["slots"])
    return dict(q=q.to(torch.bfloat16 if c["kind"] == "f32" else s["q"].dtype), k=k, v=v)


def _attention(s):
    c = s["case"]
    Hq, Hkv, D = c["q_heads"], c["kv_heads"], c["head_dim"]
    G, B = Hq // Hkv, s["lens"].shape[0]
    if own:
        out = torch.empty_like(s["q"])
        lse = torch.empty(out.shape[0], Hq, device=out.device) if c["stats"] else None
        weights = s["new_weights"] if c["stats"] else None
        s["cache"].attention(s["q"], s["cu"], s["lens"], s["table"], out, s["workspace"], max_count=c["tokens"],
                             gate=s["gate"], lse=lse, weights_in=s["weights"], weights_out=weights)
        return dict(out=out, lse=lse, weights=weights) if c["stats"] else dict(out=out)
    counts = s["cu"][1:] - s["cu"][:-1]
    n, width = c["tokens"], s["table"].shape[1] * PAGE
    j = torch.arange(n, device=s["q"].device)
    fed = j[None, :] < counts[:, None]  # [B, n]
    rows = (s["cu"][:-1, None] + j[None, :]).clamp(max=s["q"].shape[0] - 1).long()
    k, v = _values(s["pool"][s["table"].long()], D)  # [B, pages, Hkv, 16, D]
    k = k.permute(0, 2, 1, 3, 4).reshape(B, Hkv, width, D)
    v = v.permute(0, 2, 1, 3, 4).reshape(B, Hkv, width, D)
    q = s["q"][rows].float().view(B, n, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, n * G, D)
    seen = s["lens"][:, None] - counts[:, None] + j[None, :] + 1  # keys that token j sees
    seen = torch.where(fed, seen, 0)
    mask = torch.arange(width, device=q.device)[None, None, :] < seen[:, :, None]  # [B, n, width]
    mask = mask[:, None, :, None, :].expand(B, 1, n, G, width).reshape(B, 1, n * G, width)
    x = (q @ k.transpose(-1, -2) / math.sqrt(D)).masked_fill_(~mask, -math.inf)
    top = x.amax(-1, keepdim=True).clamp(min=-3e38)
    p = x.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    p /= torch.where(total > 0, total, 1.0)
    v = torch.where(torch.arange(width, device=q.device)[None, None, :, None] < s["lens"][:, None, None, None], v, 0.0)
    y = (p @ v).view(B, Hkv, n, G, D).permute(0, 2, 1, 3, 4).reshape(B, n, Hq, D)
    out = torch.empty(s["q"].shape, device=q.device)
    out[rows[fed]] = y[fed]
    if s["gate"] is not None:
        out = out * torch.sigmoid(s["gate"])
    out = out.to(s["q"].dtype)
    if not c["stats"]:
        return dict(out=out)
    lse = torch.empty(s["q"].shape[:2], device=q.device)
    lse[rows[fed]] = (top + total.log()).view(B, Hkv, n, G).permute(0, 2, 1, 3).reshape(B, n, Hq)[fed]
    # the keys of the call's own tokens start from zero
    at = torch.arange(width, device=q.device)[None, None, :]
    old = s["weights"].masked_fill((at >= (s["lens"] - counts)[:, None, None]) & (at < s["lens"][:, None, None]), 0.0)
    return dict(out=out, lse=lse, weights=old + p.sum(2))


def _evict(s):
    c = s["case"]
    D, Hkv, keep, recent = c["head_dim"], c["kv_heads"], c["keep"], c["recent"]
    B, width = s["lens"].shape[0], s["weights"].shape[-1]
    dev = s["lens"].device
    if own:
        kept = torch.empty(B, Hkv, keep, dtype=torch.int32, device=dev)
        lens = torch.empty(B, dtype=torch.int32, device=dev)
        weights = torch.empty(B, Hkv, keep, device=dev)
        s["cache"].evict(s["lens"], s["table"], s["new_table"], s["weights"], keep, recent, kept, lens, weights)
        k = torch.empty(s["slots"].shape[0], Hkv, D, dtype=torch.float32, device=dev)
        v = torch.empty_like(k)
        s["cache"].read(s["slots"], k, v)
        return dict(kept=kept, lens=lens, weights=weights, k=k, v=v)
    n = s["lens"].long()[:, None, None]
    at = torch.arange(width, device=dev)[None, None, :]
    key = s["weights"].masked_fill((at >= n - recent) & (at < n), math.inf).masked_fill(at >= n, -math.inf)
    order = key.sort(dim=-1, descending=True, stable=True).indices  # ties: the lowest index first
    new = torch.minimum(n, torch.tensor(keep, device=dev))
    wide = max(0, keep - width)
    order = torch.nn.functional.pad(order[..., :keep], (0, wide), value=width)
    j = torch.arange(keep, device=dev)[None, None, :]
    kept = torch.where(j < new, order, width).sort(-1).values
    there = j < new
    source = kept.clamp(max=width - 1)
    weights = torch.where(there, s["weights"].gather(-1, source), 0.0)
    kept = torch.where(there, kept, -1).to(torch.int32)
    # bytes of the kept keys, moved head by head
    p = _places(D, dev)
    key_bytes = torch.cat([p["k_bytes"], p["v_bytes"], (p["k_meta"][..., None] + torch.arange(4, device=dev)).flatten(1),
                           (p["v_meta"][..., None] + torch.arange(4, device=dev)).flatten(1)], 1)
    b, h, i = there.expand(B, Hkv, keep).nonzero(as_tuple=True)
    old = source[b, h, i]
    src_page, dst_page = s["table"][b, old // PAGE].long(), s["new_table"][b, i // PAGE].long()
    s["pool"][dst_page[:, None], h[:, None], key_bytes[i % PAGE]] = s["pool"][src_page[:, None], h[:, None], key_bytes[old % PAGE]]
    k, v = _cached(s["pool"], D, s["slots"])
    return dict(kept=kept, lens=new[:, 0, 0].to(torch.int32), weights=weights, k=k, v=v)


def run(state):
    return {"append": _append, "attention": _attention, "evict": _evict}[state["case"]["op"]](state)


def work(case):
    Hq, Hkv, D = case["q_heads"], case["kv_heads"], case["head_dim"]
    token = Hkv * D * 9 / 8  # a cached token's bytes in one layer: K and V nibbles, scale / bias pairs
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["op"] == "append":
        T, e = case["tokens"], size[case["kind"]]
        move = T * ((Hq + 2 * Hkv) * D * e + Hq * D * 2 + token + 12)  # rows in, queries out, cache written
        move += T * (token + 2 * Hkv * D * 4)  # the read back
        return dict(bytes=move, flops=T * (Hq + 2 * Hkv) * D * 12)
    lens = _lengths(case)
    if case["op"] == "evict":
        kept = [min(n, case["keep"]) for n in lens]
        cut = sum(n for n in lens)
        return dict(bytes=cut * Hkv * 4 + sum(kept) * (2 * token + Hkv * 8) + sum(kept) * (token + 2 * Hkv * D * 4),
                    flops=cut * Hkv * 4)
    counts = _counts(case, lens)
    pairs = sum(c * n - c * (c - 1) / 2 for c, n in zip(counts, lens))  # (query token, key) pairs
    move = sum(lens) * token + sum(counts) * Hq * D * (4 + (4 if case["gate"] else 0))
    if case["stats"]:
        move += sum(lens) * Hkv * 8 + sum(counts) * Hq * 4
    return dict(bytes=move, flops=4 * pairs * Hq * D)


# ------------------------------------------------------------------ the definitions in 64 bits

def _exact_block(block, D):
    """K and V in 64 bits of host blocks [n, 18 D] (numpy), token by token, from the page layout."""
    n = block.shape[0]
    k, v = np.zeros((n, PAGE, D)), np.zeros((n, PAGE, D))
    words = np.ascontiguousarray(block[:, :16 * D]).view("<u4")
    pair = (np.ascontiguousarray(block[:, 16 * D:]).view("<u2").astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    pair = pair.reshape(n, 2, PAGE, D // GROUP, 2)
    chunk = min(D // 32, 4)
    for t in range(PAGE):
        for w in range(D // 8):
            d = 8 * w
            grp, half, lane = d // 64, d % 64 // 32, d % 32 // 8
            i = 2 * grp + half
            word = words[:, ((i // chunk) * PAGE + t) * 4 * chunk + lane * chunk + i % chunk]
            lane = d % 64 // 8
            per = 512 // D
            other = words[:, 2 * D + ((lane // per) * PAGE + (t & 1) * 8 + t // 2) * 8 + lane % per * (D // 64) + grp]
            for e in range(8):
                k[:, t, d + e] = (word >> (4 * (e // 2) + 16 * (e % 2))) & 15
                v[:, t, d + e] = (other >> (4 * e)) & 15
    scale, bias = pair[..., 0].repeat(GROUP, -1), pair[..., 1].repeat(GROUP, -1)
    return k * scale[:, 0] + bias[:, 0], v * scale[:, 1] + bias[:, 1]


def _exact_tokens(s, case, table, length):
    """K and V [KV head, length, D] in 64 bits, on the GPU, of one sequence."""
    pool = s["pool"][table[: -(-length // PAGE)].long()].cpu().numpy()
    n, H, _ = pool.shape
    k, v = _exact_block(pool.reshape(n * H, -1), case["head_dim"])
    put = lambda x: torch.from_numpy(x.reshape(n, H, PAGE, -1)).cuda().permute(1, 0, 2, 3).reshape(H, n * PAGE, -1)[:, :length]  # noqa: E731
    return put(k), put(v)


def exact(case, seed):
    s = prepare(case, seed)
    Hq, Hkv, D = case["q_heads"], case["kv_heads"], case["head_dim"]
    G = Hq // Hkv
    if case["op"] == "append":
        got = {}
        pos = s["positions"].cpu().numpy().astype(np.float64)
        for name in "qkv":
            x = s[name].double().cpu().numpy()
            if name != "v":
                w = s[name + "_norm"].double().cpu().numpy()
                x = x / np.sqrt(np.mean(x ** 2, -1, keepdims=True) + EPS) * w
                r = case["rope"]
                for j in range(r // 2):
                    angle = (pos * THETA ** (-2.0 * j / r))[:, None]
                    z = (x[..., j] + 1j * x[..., j + r // 2]) * np.exp(1j * angle)
                    x[..., j], x[..., j + r // 2] = z.real, z.imag
            if name != "q":
                g = torch.from_numpy(x.reshape(*x.shape[:2], D // GROUP, GROUP))
                step = ((g.max(-1).values - g.min(-1).values) / 15).to(torch.float32).to(torch.bfloat16).double()[..., None]
                base = g.min(-1).values.to(torch.float32).to(torch.bfloat16).double()[..., None]
                x = (((g - base) / step).round().clamp(0, 15) * step + base).reshape(x.shape).numpy()
            got[name] = x
        return got
    if case["op"] == "evict":
        ks, vs, kept_all = [], [], []
        lens, weights = s["lens"].tolist(), s["weights"].cpu().numpy()
        out_w = np.zeros((len(lens), Hkv, case["keep"]))
        if sum(lens) > 150_000:
            return None
        for b, n in enumerate(lens):
            k, v = _exact_tokens(s, case, s["table"][b], n)
            m, recent = min(n, case["keep"]), min(n, case["recent"])
            rows_k, rows_v = [], []
            for h in range(Hkv):
                if n > case["keep"]:
                    old = weights[b, h, : n - recent]
                    best = np.lexsort((np.arange(n - recent), -old))[: m - recent]
                    idx = np.concatenate([np.sort(best), np.arange(n - recent, n)])
                else:
                    idx = np.arange(n)
                out_w[b, h, :m] = weights[b, h, idx]
                at = torch.from_numpy(idx).cuda()
                rows_k.append(k[h, at])
                rows_v.append(v[h, at])
            ks.append(torch.stack(rows_k, 1))
            vs.append(torch.stack(rows_v, 1))
        return dict(kept=None, lens=None, weights=out_w, k=torch.cat(ks), v=torch.cat(vs))
    cu, lens = s["cu"].tolist(), s["lens"].tolist()
    if sum(lens) > 500_000:
        return None
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    weights = s["weights"].double() if case["stats"] else None
    for b, n in enumerate(lens):
        k, v = _exact_tokens(s, case, s["table"][b], n)
        a, z = cu[b], cu[b + 1]
        for h in range(Hq):
            x = s["q"][a:z, h].double() @ k[h // G].T * D ** -0.5
            late = torch.arange(n, device="cuda")[None, :] > (n - (z - a) + torch.arange(z - a, device="cuda"))[:, None]
            x[late] = -math.inf
            p = torch.softmax(x, -1)
            out[a:z, h] = p @ v[h // G]
            lse[a:z, h] = torch.logsumexp(x, -1)
            if weights is not None:
                if h % G == 0:
                    weights[b, h // G, n - (z - a):n] = 0
                weights[b, h // G, :n] += p.sum(0)
    if s["gate"] is not None:
        out *= torch.sigmoid(s["gate"].double())
    return dict(out=out, lse=lse, weights=weights) if case["stats"] else dict(out=out)
