"""Plain 64-bit forms of the 4-bit KV-cache operators for the tests: the
quantiser, the append's norm and rotation, attention over given values and the
eviction rule, each from its definition and without the page layout."""
import math

import torch

PAGE, GROUP = 16, 64


def quantised(x):
    """The values that stand for x [..., D] (64 bits) after 4-bit storage, and per value the largest
    magnitude its group can store (|bias| + 15 scale)."""
    g = x.double().unflatten(-1, (-1, GROUP))
    fine = torch.isfinite(g).all(-1, keepdim=True)
    z = torch.where(fine, g, 0.0)
    scale = ((z.amax(-1, keepdim=True) - z.amin(-1, keepdim=True)) / 15).float().bfloat16().double()
    bias = z.amin(-1, keepdim=True).float().bfloat16().double()
    n = torch.where(scale > 0, ((z - bias) / torch.where(scale > 0, scale, 1.0)).round().clamp(0, 15), 0.0)
    # the sum is rounded once to 32 bits
    y = torch.where(fine, (scale * n + bias).float().double(), math.nan)
    return y.flatten(-2), (bias.abs() + 15 * scale).expand_as(g).flatten(-2)


def normed_rotated(x, positions, norm=None, eps=1e-6, theta=1e7, rope=0):
    """RMSNorm and partial rotation of [T, H, D] in 64 bits."""
    x = x.double()
    if norm is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * norm.double()
    if rope:
        j = torch.arange(rope // 2, device=x.device, dtype=torch.float64)
        angle = positions.double()[:, None, None] * theta ** (-2 * j / rope)
        a, b = x[..., :rope // 2], x[..., rope // 2:rope]
        x = torch.cat([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos(), x[..., rope:]], -1)
    return x


def attention(q, k, v, most_k, scale):
    """One sequence: q [n, Hq, D], k / v [L, Hkv, D] in 64 bits (the values in the cache), causal bottom-right.
    Returns (out, lse, weights [Hkv, L], error of a logit by 32-bit sums [n, Hq])."""
    n, Hq, D = q.shape
    L, Hkv, _ = k.shape
    G = Hq // Hkv
    q, k, v = q.double(), k.double(), v.double()
    kk, vv = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    x = torch.einsum("nhd,lhd->hnl", q, kk) * scale
    late = torch.arange(L, device=q.device)[None, :] > (L - n + torch.arange(n, device=q.device))[:, None]
    x = x.masked_fill(late[None], -math.inf)
    p = torch.softmax(x, -1)
    p = torch.where(late[None].all(-1, keepdim=True), 0.0, p)
    out = torch.einsum("hnl,lhd->nhd", p, vv)
    lse = torch.logsumexp(x, -1).T
    weights = p.view(Hkv, G, n, L).sum((1, 2))
    if L:
        mass = torch.einsum("nhd,hd->nh", q.abs(), most_k.double().amax(0).repeat_interleave(G, 0))
    else:
        mass = torch.zeros(n, Hq, device=q.device, dtype=torch.float64)
    return out, lse, weights, D * 2.0 ** -23 * scale * mass


def evicted(weights, length, keep, recent):
    """Indices that stay of one (sequence, KV head), ascending: IEEE total order, lowest index on ties."""
    if length <= keep:
        return list(range(length))
    bits = weights[: length - recent].float().cpu().contiguous().view(torch.int32).tolist()
    key = []
    for b in bits:
        u = b & 0xFFFFFFFF
        key.append((~u & 0xFFFFFFFF) if u >> 31 else u | 0x80000000)
    best = sorted(range(len(key)), key=lambda i: (-key[i], i))[: keep - recent]
    return sorted(best) + list(range(length - recent, length))


class Sequences:
    """A cache of ragged sequences with the values that it stands for, on shuffled pages of a pool whose unused
    bytes are 0xFF (unused tokens then read as NaN)."""

    def __init__(self, pkg, lens, heads, seed=0, extra_pages=0, spread=1.0, pad_columns=2):
        self.Hq, self.Hkv, self.D = heads
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.gen, self.lens = gen, list(lens)
        need = [-(-n // PAGE) for n in lens]
        pages = sum(need) + extra_pages + 3
        self.pool = torch.full((pages * pkg.kv4_page_bytes(self.Hkv, self.D),), 255, dtype=torch.uint8, device="cuda")
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.cache = pkg.Kv4Cache(self.pool, self.Hq, self.Hkv, self.D, status=self.status)
        ids = torch.randperm(pages, generator=gen, device="cuda").int().tolist()
        self.spare = ids[sum(need):]
        self.table = torch.full((len(lens), max(need + [0]) + pad_columns), -1, dtype=torch.int32, device="cuda")
        self.k, self.v, self.most, at = [], [], [], 0
        for s, n in enumerate(lens):
            self.table[s, :need[s]] = torch.tensor(ids[at:at + need[s]], dtype=torch.int32)
            at += need[s]
            k = torch.randn(n, self.Hkv, self.D, generator=gen, device="cuda") * spread
            v = torch.randn(n, self.Hkv, self.D, generator=gen, device="cuda")
            if n:
                self.cache.append(None, k, v, None, self.slots(s, 0, n), None)
            qk, most = quantised(k)
            self.k.append(qk)
            self.v.append(quantised(v)[0])
            self.most.append(most)
        self.kv_lens = torch.tensor(self.lens, dtype=torch.int32, device="cuda")

    def slots(self, s, first, last):
        p = torch.arange(first, last, device="cuda")
        return self.table[s, p // PAGE].long() * PAGE + p % PAGE

    def queries(self, counts, dtype, pad=0):
        cu = [0]
        for c in counts:
            cu.append(cu[-1] + c)
        q = torch.randn(cu[-1] + pad, self.Hq, self.D, generator=self.gen, device="cuda").to(dtype)
        return q, torch.tensor(cu, dtype=torch.int32, device="cuda"), cu


def check_attention(seqs, q, cu, out, lse=None, weights=None, weights_in=None, gate=None, scale=None):
    """Every output of one attention call against the 64-bit form. Tolerances, from the number formats: a logit
    is a 32-bit sum (ds, from attention()); the softmax weights times a value's step are rounded to fp16 (half a
    step: 2^-11 of at most 15 steps of the value's group, i.e. of the range it spans); the exponential and the
    sigmoid have a relative error below 2^-18; the result is rounded once to its type. Without lse and weights a
    sequence of more than 32 query rows per KV head goes through fp16 operands of K and V: each value is off by at
    most half a step, 2^-11 of it, so a logit by 2^-11 of the sum of |q| |k| (ds is D 2^-23 of it: 2^12 / D times as
    much) and an output by 2^-11 of the largest value."""
    scale = scale or seqs.D ** -0.5
    G = seqs.Hq // seqs.Hkv
    half_step = torch.finfo(out.dtype).eps / 2
    for s, n in enumerate(seqs.lens):
        a, z = cu[s], cu[s + 1]
        k, v = seqs.k[s], seqs.v[s]
        ref, ref_lse, ref_w, ds = attention(q[a:z], k, v, seqs.most[s], scale)
        vmax = v.abs().amax().item() if n else 0.0
        chunk = lse is None and weights is None and (z - a) * G > 32 and out.dtype == torch.bfloat16
        if chunk:
            ds = ds * (1 + 2.0 ** 12 / seqs.D)
        loose = 2.0 ** -11 * (3 if chunk else 2) * vmax + (2 * ds[..., None] + 2.0 ** -18) * vmax
        if gate is not None:
            sg = torch.sigmoid(gate[a:z].double())
            ref, loose = ref * sg, loose * sg + ref.abs() * 2.0 ** -18
        tol = half_step * (ref.abs() + loose) + loose + torch.finfo(out.dtype).tiny * torch.finfo(out.dtype).eps
        bad = (out[a:z].double() - ref).abs() > tol
        assert not bad.any(), (s, n, z - a, (out[a:z].double() - ref).abs().max().item())
        assert not torch.isnan(out[a:z]).any()
        if lse is not None:
            fin = torch.isfinite(ref_lse)
            assert torch.equal(fin, torch.isfinite(lse[a:z])) and (lse[a:z][~fin] < 0).all()
            d = (lse[a:z].double() - ref_lse).abs()[fin]
            assert (d <= (ds + 2.0 ** -18 + 2.0 ** -22 * ref_lse.abs())[fin]).all(), d.max()
        if weights is not None and n:
            old = torch.zeros(seqs.Hkv, n, dtype=torch.float64, device="cuda")
            if weights_in is not None:
                keep = max(0, n - (z - a))
                old[:, :keep] = weights_in[s, :, :keep].double()
            want = old + ref_w
            slack = (2 * ds.max().item() if z > a else 0) + 2.0 ** -18 + (z - a) * G * 2.0 ** -23
            d = (weights[s, :, :n].double() - want).abs()
            assert (d <= slack * ref_w + 2.0 ** -22 * want + 1e-30).all(), d.max()
