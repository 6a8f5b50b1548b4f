"""The 4-bit KV-cache operators on the GPU against their 64-bit forms
(kv4_util.py), at the sizes, masks, strides and streams where they can go wrong,
and a run of them together as a serving loop makes it."""
import math

import pytest

from conftest import has_cuda

pytestmark = pytest.mark.gpu

if has_cuda():
    import torch

    import kv4_util as U
    from kv4_util import Sequences, check_attention, quantised

HEADS = [(4, 1, 64), (16, 2, 256), (20, 4, 128)]


@pytest.fixture(autouse=True)
def _cuda():
    if not has_cuda():
        pytest.skip("no CUDA device")


def new_cache(pkg, heads, pages, fill=255):
    Hq, Hkv, D = heads
    pool = torch.full((pages * pkg.kv4_page_bytes(Hkv, D),), fill, dtype=torch.uint8, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    return pkg.Kv4Cache(pool, Hq, Hkv, D, status=status)


def read(cache, slots, dtype=None):
    dtype = dtype or torch.float32
    k = torch.empty(slots.shape[0], cache.kv_heads, cache.head_dim, dtype=dtype, device="cuda")
    v = torch.empty_like(k)
    cache.read(slots, k, v)
    return k, v


# ------------------------------------------------------------------ append and read

def rows(kind, layout, T, heads, gen):
    Hq, Hkv, D = heads
    dtype = getattr(torch, kind)
    if layout == "plain":
        return [torch.randn(T, h, D, generator=gen, device="cuda").to(dtype) for h in (Hq, Hkv, Hkv)]
    # views of one projection row [query, gate] x Hq, keys, values; "odd" rows start at odd elements
    width = (2 * Hq + 2 * Hkv) * D + (3 if layout == "odd" else 0)
    row = torch.randn(T, width, generator=gen, device="cuda").to(dtype)
    at = 1 if layout == "odd" else 0
    q = row[:, at:at + 2 * Hq * D].unflatten(1, (Hq, 2, D))[:, :, 0]
    at += 2 * Hq * D
    return [q, row[:, at:at + Hkv * D].unflatten(1, (Hkv, D)), row[:, at + Hkv * D:at + 2 * Hkv * D].unflatten(1, (Hkv, D))]


@pytest.mark.parametrize("T", [1, 33])
@pytest.mark.parametrize("layout", ["plain", "fused", "odd"])
@pytest.mark.parametrize("kind", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("heads,rope", [((4, 1, 64), 16), ((16, 2, 256), 64), ((20, 4, 128), 128), ((6, 6, 64), 0), ((3, 1, 128), 2),
                                        ((2, 2, 256), 250)])
def test_append_stores_the_quantised_rows(pkg, heads, rope, kind, layout, T):
    Hq, Hkv, D = heads
    gen = torch.Generator(device="cuda").manual_seed(T * 7 + rope)
    cache = new_cache(pkg, heads, 9)
    q, k, v = rows(kind, layout, T, heads, gen)
    pos = torch.randint(0, 40000, (T,), generator=gen, device="cuda", dtype=torch.int32)
    slots = torch.randperm(9 * 16, generator=gen, device="cuda")[:T].contiguous()
    qn = 1 + 0.2 * torch.randn(D, generator=gen, device="cuda")
    kn = 1 + 0.2 * torch.randn(D, generator=gen, device="cuda")
    for out_kind in ("float32", "float16", "bfloat16"):
        out = torch.empty(T, Hq, D, dtype=getattr(torch, out_kind), device="cuda")
        cache.append(q, k, v, pos, slots, out, q_norm=qn, k_norm=kn, epsilon=1e-6, theta=1e6, rope_dims=rope)
        want = U.normed_rotated(q, pos, qn, 1e-6, 1e6, rope)
        # 32-bit norm: a sum of D squares (relative error D 2^-24 at most, halved by the root), four further
        # roundings and the root's own 2^-22; a rotated value adds its partner's error
        size = want.abs() + (want.abs().amax(-1, keepdim=True) if rope else 0)
        tol = torch.finfo(out.dtype).eps / 2 * want.abs() + (D / 2 + 12) * 2.0 ** -24 * size + torch.finfo(out.dtype).tiny * torch.finfo(out.dtype).eps
        assert ((out.double() - want).abs() <= tol * (1 + 2.0 ** -8)).all()
    got_k, got_v = read(cache, slots)
    want_k, want_v = quantised(U.normed_rotated(k, pos, kn, 1e-6, 1e6, rope))[0], quantised(v)[0]
    assert torch.equal(got_k.double(), want_k) and torch.equal(got_v.double(), want_v)
    for dtype in (torch.float16, torch.bfloat16):  # read rounds once
        k16, v16 = read(cache, slots, dtype)
        assert torch.equal(k16, want_k.float().to(dtype)) and torch.equal(v16, want_v.float().to(dtype))
    cache.check()


def test_append_leaves_other_tokens_alone(pkg):
    heads = (4, 2, 64)
    cache = new_cache(pkg, heads, 3)
    gen = torch.Generator(device="cuda").manual_seed(1)
    all_slots = torch.arange(48, device="cuda")
    k = torch.randn(48, 2, 64, generator=gen, device="cuda")
    v = torch.randn(48, 2, 64, generator=gen, device="cuda")
    cache.append(None, k, v, None, all_slots, None)
    before = read(cache, all_slots)
    fresh = torch.randn(3, 2, 64, generator=gen, device="cuda")
    slots = torch.tensor([17, -1, 46], device="cuda")
    cache.append(None, fresh, fresh, None, slots, None)
    after = read(cache, all_slots)
    same = torch.ones(48, dtype=torch.bool, device="cuda")
    same[[17, 46]] = False
    for a, b, x in zip(before, after, (fresh, fresh)):
        assert torch.equal(a[same], b[same])
        assert torch.equal(b[[17, 46]].double(), quantised(x[[0, 2]])[0])
    cache.check()


def test_append_queries_only_and_without_norm(pkg):
    cache = new_cache(pkg, (4, 2, 64), 1, fill=7)
    q = torch.randn(5, 4, 64, device="cuda")
    out = torch.empty_like(q)
    before = cache.pool.clone()
    cache.append(q, None, None, None, None, out)
    assert torch.equal(out, q) and torch.equal(cache.pool, before)


def test_append_special_values(pkg):
    """Constant groups, groups of one sign, infinities and NaN, tiny and huge values."""
    cache = new_cache(pkg, (1, 1, 128), 1)
    x = torch.randn(8, 1, 128, device="cuda")
    x[0] = 0.0
    x[1] = 3.140625  # a bf16 value: stored exactly
    x[2, :, :64] = math.inf
    x[3, :, 70] = math.nan
    x[4] = x[4].abs() * 1e-30
    x[5] = x[5] * 1e30
    x[6, :, :64] = -math.inf
    x[7] = x[7].abs() + 100
    slots = torch.arange(8, device="cuda")
    cache.append(None, x, x, None, slots, None)
    want = quantised(x)[0]
    for got in read(cache, slots):
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got.double().nan_to_num(), want.nan_to_num())
        assert torch.isnan(got[2, :, :64]).all() and torch.isnan(got[3, :, 64:]).all() and torch.isnan(got[6, :, :64]).all()
        assert not torch.isnan(got[2, :, 64:]).any()
        assert (got[0] == 0).all() and (got[1] == 3.140625).all()


def test_append_halfway_values_round_to_even(pkg):
    """Group 0, 1, .., 15 and halves: scale 1, bias 0, so n + 1/2 is a tie."""
    cache = new_cache(pkg, (1, 1, 64), 1)
    x = torch.zeros(1, 1, 64, device="cuda")
    x[0, 0, :16] = torch.arange(16, device="cuda")
    x[0, 0, 16:31] = torch.arange(15, device="cuda") + 0.5
    cache.append(None, x, x, None, torch.zeros(1, dtype=torch.int64, device="cuda"), None)
    k, v = read(cache, torch.zeros(1, dtype=torch.int64, device="cuda"))
    assert torch.equal(k, x.round()) and torch.equal(v, x.round())


def test_slots_out_of_range_are_skipped_and_reported(pkg):
    cache = new_cache(pkg, (2, 1, 64), 2, fill=0)
    x = torch.randn(3, 1, 64, device="cuda")
    slots = torch.tensor([5, 32, 1 << 40], device="cuda")
    cache.append(None, x, x, None, slots, None)
    with pytest.raises(pkg.NativeError, match="flag 2"):
        cache.check()
    cache.check()  # cleared
    k, _ = read(cache, torch.tensor([5, -1, 31], device="cuda"))
    assert torch.equal(k[:1].double(), quantised(x[:1])[0]) and not k[1:].any()
    k, v = read(cache, slots)
    assert not k[1:].any() and not v[1:].any()
    with pytest.raises(pkg.NativeError, match="flag 2"):
        cache.check()


# ------------------------------------------------------------------ attention

def attend(pkg, seqs, q, cu, counts, stats=False, weights_in=None, gate=None, fill=None, **kw):
    out = torch.full_like(q, 77.0)
    ws = torch.empty(seqs.cache.workspace_bytes(len(counts), max(1, q.shape[0])), dtype=torch.uint8, device="cuda")
    lse = torch.full(q.shape[:2], 77.0, device="cuda") if stats else None
    weights = None
    if stats:
        weights = torch.full((len(counts), seqs.Hkv, seqs.table.shape[1] * 16), 55.0, device="cuda")
    seqs.cache.attention(q, cu, seqs.kv_lens, seqs.table, out, ws, max(1, max(counts)), gate=gate, lse=lse,
                         weights_in=weights_in, weights_out=weights, **kw)
    return out, lse, weights


@pytest.mark.parametrize("kind", ["float16", "bfloat16"])
@pytest.mark.parametrize("heads", HEADS + [(6, 6, 64), (15, 3, 128), (16, 1, 64), (9, 1, 256), (32, 2, 128)])
def test_decode(pkg, heads, kind):
    lens = [1, 2, 15, 16, 17, 31, 33, 64, 100, 257, 700]
    seqs = Sequences(pkg, lens, heads, seed=3)
    counts = [1] * len(lens)
    q, cu, host = seqs.queries(counts, getattr(torch, kind))
    gate = torch.randn(q.shape, generator=seqs.gen, device="cuda")
    out, lse, weights = attend(pkg, seqs, q, cu, counts, stats=True, gate=gate)
    check_attention(seqs, q, host, out, lse, weights, gate=gate)
    plain, _, _ = attend(pkg, seqs, q, cu, counts)
    check_attention(seqs, q, host, plain)
    for s, n in enumerate(lens):  # columns behind the length keep what they held
        assert (weights[s, :, n:] == 55).all()
    seqs.cache.check()


@pytest.mark.parametrize("counts,lens", [
    ([0, 3, 1, 0, 7, 2], [5, 3, 40, 0, 9, 100]), ([4, 4, 4], [4, 17, 500]), ([17, 1, 130], [17, 300, 161]),
    ([200], [200]), ([64, 33], [1000, 33]), ([129], [640]), ([0, 0, 1], [0, 16, 1])])
@pytest.mark.parametrize("heads", HEADS + [(5, 1, 64), (32, 2, 256)])
def test_ragged_counts(pkg, heads, counts, lens):
    seqs = Sequences(pkg, lens, heads, seed=5)
    q, cu, host = seqs.queries(counts, torch.bfloat16, pad=3)
    width = seqs.table.shape[1] * 16
    win = torch.rand(len(lens), seqs.Hkv, width, generator=seqs.gen, device="cuda")
    out, lse, weights = attend(pkg, seqs, q, cu, counts, stats=True, weights_in=win)
    check_attention(seqs, q, host, out, lse, weights, weights_in=win)
    plain, _, _ = attend(pkg, seqs, q, cu, counts)
    check_attention(seqs, q, host, plain)
    assert (plain[host[-1]:] == 77).all()
    assert (out[host[-1]:] == 77).all() and (lse[host[-1]:] == 77).all()  # rows behind the last sequence
    for s, n in enumerate(lens):
        assert (weights[s, :, n:] == 55).all()
    seqs.cache.check()


@pytest.mark.parametrize("heads", HEADS)
def test_rows_that_see_no_key(pkg, heads):
    """More query tokens than cached keys: the first ones see nothing."""
    lens, counts = [3, 0, 20], [5, 2, 24]
    seqs = Sequences(pkg, lens, heads, seed=9)
    q, cu, host = seqs.queries(counts, torch.float16)
    out, lse, weights = attend(pkg, seqs, q, cu, counts, stats=True)
    check_attention(seqs, q, host, out, lse, weights)
    plain, _, _ = attend(pkg, seqs, q, cu, counts)
    check_attention(seqs, q, host, plain)
    for row in (0, 1, 5, 6, 7, 8, 9, 10):
        assert (out[row] == 0).all() and (lse[row] == -math.inf).all() and (plain[row] == 0).all()


@pytest.mark.parametrize("spread,scale", [(30.0, 0.0), (1.0, 8.0), (1e-4, 0.25), (3e4, 1e-6)])
@pytest.mark.parametrize("heads", HEADS)
def test_large_and_small_logits(pkg, heads, spread, scale):
    seqs = Sequences(pkg, [40, 700], heads, seed=11, spread=spread)
    q, cu, host = seqs.queries([1, 3], torch.bfloat16)
    out, lse, weights = attend(pkg, seqs, q, cu, [1, 3], stats=True, scale=scale)
    check_attention(seqs, q, host, out, lse, weights, scale=scale)
    q, cu, host = seqs.queries([30, 70], torch.float16)
    out, _, _ = attend(pkg, seqs, q, cu, [30, 70], scale=scale)
    check_attention(seqs, q, host, out, scale=scale)


@pytest.mark.parametrize("size", [1e-6, 1e-3, 1e3, 1e30])
def test_values_of_any_size(pkg, size):
    """V far outside fp16, beside values of ordinary size."""
    heads = (8, 1, 128)
    seqs = Sequences(pkg, [200, 50], heads, seed=12)
    for s, n in enumerate(seqs.lens):
        v = torch.randn(n, 1, 128, generator=seqs.gen, device="cuda")
        v[:, :, 64:] *= size
        v[n // 2:] *= 1e-3
        zero = torch.zeros(n, 1, 128, device="cuda")
        seqs.cache.append(None, zero, v, None, seqs.slots(s, 0, n), None)
        seqs.k[s], seqs.most[s] = quantised(zero)
        seqs.v[s] = quantised(v)[0]
    q, cu, host = seqs.queries([1, 2], torch.bfloat16)
    out, _, _ = attend(pkg, seqs, q, cu, [1, 2])
    for a, z in ((0, 64), (64, 128)):  # each group by its own size
        part = Sequences.__new__(Sequences)
        part.__dict__.update(seqs.__dict__)
        for s in range(2):
            n = seqs.lens[s]
            ref, _, _, _ = U.attention(q[host[s]:host[s + 1]], seqs.k[s], seqs.v[s], seqs.most[s], 128 ** -0.5)
            got, want = out[host[s]:host[s + 1], :, a:z].double(), ref[..., a:z]
            vmax = seqs.v[s][..., a:z].abs().max().item()
            # zero keys: equal weights; their product with a step rounds to fp16, the result to bf16
            assert ((got - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -10 + 2.0 ** -17) * vmax).all(), (s, a)


def test_queries_of_any_size(pkg):
    """Rows far outside fp16 (bf16 queries) and zero rows; a row with a NaN or infinity gives NaN and only there."""
    heads = (8, 1, 128)
    seqs = Sequences(pkg, [100], heads, seed=13)
    q, cu, host = seqs.queries([1], torch.bfloat16)
    q[0, 0] *= 1e30
    q[0, 1] = 0
    q[0, 2] *= 1e-30
    q[0, 3] *= 1e5
    clean = q.clone()
    scale = 1e-6
    out, _, _ = attend(pkg, seqs, q, cu, [1], scale=scale)
    ref, _, _, ds = U.attention(clean, seqs.k[0], seqs.v[0], seqs.most[0], scale)
    vmax = seqs.v[0].abs().max()
    for h in range(1, 8):
        tol = 2.0 ** -8 * ref[0, h].abs() + (2.0 ** -10 + 2 * ds[0, h] + 2.0 ** -17) * vmax
        assert ((out[0, h].double() - ref[0, h]).abs() <= tol).all(), h
    assert torch.isfinite(out).all()  # one key takes everything in head 0
    q[0, 4, 5] = math.nan
    q[0, 6, 7] = math.inf
    again, _, _ = attend(pkg, seqs, q, cu, [1], scale=scale)
    assert torch.isnan(again[0, 4]).all() and torch.isnan(again[0, 6]).all()
    keep = [0, 1, 2, 3, 5, 7]
    assert torch.equal(again[0, keep], out[0, keep])


def test_nan_in_the_cache_reaches_only_its_own_rows(pkg):
    """A NaN key makes the rows that see it NaN; the sequence beside it and rows before it are untouched."""
    heads = (4, 2, 64)
    seqs = Sequences(pkg, [20, 30], heads, seed=14)
    q, cu, host = seqs.queries([4, 2], torch.float16)
    good, _, _ = attend(pkg, seqs, q, cu, [4, 2])
    bad = torch.full((1, 2, 64), math.nan, device="cuda")
    slot = seqs.slots(0, 18, 19)
    k_old, v_old = read(seqs.cache, slot)
    seqs.cache.append(None, bad, v_old, None, slot, None)
    out, _, _ = attend(pkg, seqs, q, cu, [4, 2])
    assert torch.equal(out[:2], good[:2]) and torch.equal(out[4:], good[4:])  # tokens 0, 1 see keys 0..17
    assert torch.isnan(out[2:4]).all()


def test_nan_value_reaches_only_the_rows_that_see_it(pkg):
    seqs = Sequences(pkg, [20], (4, 2, 64), seed=26)
    q, cu, host = seqs.queries([4], torch.float16)
    good, _, _ = attend(pkg, seqs, q, cu, [4])
    slot = seqs.slots(0, 18, 19)
    k_old, _ = read(seqs.cache, slot)
    seqs.cache.append(None, k_old, torch.full((1, 2, 64), math.inf, device="cuda"), None, slot, None)
    out, _, _ = attend(pkg, seqs, q, cu, [4])
    assert torch.equal(out[:2], good[:2]) and torch.isnan(out[2:]).all()


def test_more_rows_than_max_count_are_reported(pkg):
    seqs = Sequences(pkg, [20, 20], (4, 2, 64), seed=27)
    q, cu, host = seqs.queries([4, 2], torch.float16)
    want, _, _ = attend(pkg, seqs, q, cu, [4, 2])
    seqs.cache.check()
    out, _, _ = attend(pkg, seqs, q, cu, [2, 2])  # claims two rows at most
    assert torch.equal(out[4:], want[4:]) and (out[:4] == 77).all()
    with pytest.raises(pkg.NativeError, match="flag 2"):
        seqs.cache.check()


def test_strided_queries_and_outputs(pkg):
    heads = (8, 2, 128)
    seqs = Sequences(pkg, [50, 7, 200], heads, seed=15)
    counts = [1, 2, 5]
    q, cu, host = seqs.queries(counts, torch.bfloat16)
    want, _, _ = attend(pkg, seqs, q, cu, counts)
    T = q.shape[0]
    ws = torch.empty(seqs.cache.workspace_bytes(3, T), dtype=torch.uint8, device="cuda")
    for lead, tail in ((0, 0), (1, 2), (8, 8)):  # odd starts too
        buf = torch.zeros(T, 8 * 2 * 128 + lead + tail, dtype=torch.bfloat16, device="cuda")
        view = buf[:, lead:lead + 2048].unflatten(1, (8, 2, 128))[:, :, 1]
        view.copy_(q)
        outs = torch.full((8, T, 128 + lead), 3.0, dtype=torch.bfloat16, device="cuda")
        out = outs[:, :, lead:].transpose(0, 1)
        seqs.cache.attention(view, cu, seqs.kv_lens, seqs.table, out, ws, 5)
        assert torch.equal(out, want)
        assert (outs[:, :, :lead] == 3).all()


def test_pages_out_of_range_count_as_absent(pkg):
    heads = (16, 2, 256)
    seqs = Sequences(pkg, [40, 40], heads, seed=16)
    counts = [2, 2]
    q, cu, host = seqs.queries(counts, torch.bfloat16)
    seqs.table[0, 1] = 1 << 20
    seqs.table[1, 0] = -7
    out, _, _ = attend(pkg, seqs, q, cu, counts)
    with pytest.raises(pkg.NativeError, match="flag 2"):
        seqs.cache.check()
    gone = [range(16, 32), range(0, 16)]
    for s in range(2):
        keep = [i for i in range(40) if i not in gone[s]]
        ref, _, _, ds = U.attention(q[2 * s:2 * s + 2], seqs.k[s][keep], seqs.v[s][keep], seqs.most[s][keep], 1 / 16)
        vmax = seqs.v[s].abs().max()
        tol = 2.0 ** -8 * ref.abs() + (2.0 ** -10 + 2 * ds[..., None] + 2.0 ** -17) * vmax
        assert ((out[2 * s:2 * s + 2].double() - ref).abs() <= tol).all()


def test_lengths_beyond_the_table_are_cut_and_reported(pkg):
    seqs = Sequences(pkg, [32, 16], (4, 1, 64), seed=17, pad_columns=0)
    q, cu, host = seqs.queries([1, 1], torch.float16)
    want, _, _ = attend(pkg, seqs, q, cu, [1, 1])
    seqs.cache.check()
    seqs.kv_lens = torch.tensor([1 << 30, 16], dtype=torch.int32, device="cuda")
    out, _, _ = attend(pkg, seqs, q, cu, [1, 1])
    assert torch.equal(out, want)
    with pytest.raises(pkg.NativeError, match="flag 2"):
        seqs.cache.check()
    seqs.kv_lens = torch.tensor([-5, 16], dtype=torch.int32, device="cuda")
    out, _, _ = attend(pkg, seqs, q, cu, [1, 1])
    assert torch.equal(out[1], want[1]) and (out[0] == 0).all()
    with pytest.raises(pkg.NativeError, match="flag 2"):
        seqs.cache.check()


def test_offsets_past_32_bits(pkg):
    """A pool of more than 4 GiB with the sequence on its last pages."""
    heads = (16, 2, 256)
    page = pkg.kv4_page_bytes(2, 256)
    pages = (1 << 32) // page + 40
    pool = torch.empty(pages * page, dtype=torch.uint8, device="cuda")
    cache = pkg.Kv4Cache(pool, *heads)
    ids = torch.arange(pages - 20, pages, device="cuda", dtype=torch.int32)[None].contiguous()
    k = torch.randn(300, 2, 256, device="cuda")
    v = torch.randn(300, 2, 256, device="cuda")
    p = torch.arange(300, device="cuda")
    slots = ids[0, p // 16].long() * 16 + p % 16
    cache.append(None, k, v, None, slots, None)
    got_k, got_v = read(cache, slots)
    assert torch.equal(got_k.double(), quantised(k)[0]) and torch.equal(got_v.double(), quantised(v)[0])
    q = torch.randn(2, 16, 256, device="cuda").to(torch.bfloat16)
    seqs = Sequences.__new__(Sequences)
    seqs.Hq, seqs.Hkv, seqs.D, seqs.lens, seqs.cache, seqs.table = 16, 2, 256, [300], cache, ids
    seqs.kv_lens = torch.tensor([300], dtype=torch.int32, device="cuda")
    seqs.k, seqs.v, seqs.most = [quantised(k)[0]], [quantised(v)[0]], [quantised(k)[1]]
    cu = torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    out, _, _ = attend(pkg, seqs, q, cu, [2])
    check_attention(seqs, q, [0, 2], out)


def test_same_inputs_same_bits(pkg):
    seqs = Sequences(pkg, [5000, 17, 300, 2000], (16, 2, 256), seed=18)
    counts = [1, 3, 40, 1]
    q, cu, _ = seqs.queries(counts, torch.bfloat16)
    first = attend(pkg, seqs, q, cu, counts, stats=True)
    for _ in range(3):
        again = attend(pkg, seqs, q, cu, counts, stats=True)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_many_sequences(pkg):
    """More sequences than multiprocessors, most of them short."""
    lens = [1 + (i * 37) % 90 for i in range(700)]
    seqs = Sequences(pkg, lens, (4, 1, 64), seed=19)
    counts = [1] * 700
    q, cu, host = seqs.queries(counts, torch.float16)
    out, lse, weights = attend(pkg, seqs, q, cu, counts, stats=True)
    check_attention(seqs, q, host, out, lse, weights)


def test_long_decode(pkg):
    seqs = Sequences(pkg, [30011, 9000], (16, 2, 256), seed=20)
    q, cu, host = seqs.queries([1, 1], torch.float16)
    out, lse, weights = attend(pkg, seqs, q, cu, [1, 1], stats=True)
    check_attention(seqs, q, host, out, lse, weights)


def test_long_chunk(pkg):
    seqs = Sequences(pkg, [2500, 700], (16, 2, 256), seed=21)
    counts = [700, 513]
    q, cu, host = seqs.queries(counts, torch.bfloat16)
    gate = torch.randn(q.shape, generator=seqs.gen, device="cuda")
    out, lse, weights = attend(pkg, seqs, q, cu, counts, stats=True, gate=gate)
    check_attention(seqs, q, host, out, lse, weights, gate=gate)
    out, _, _ = attend(pkg, seqs, q, cu, counts, gate=gate)
    check_attention(seqs, q, host, out, gate=gate)


@pytest.mark.parametrize("kind", ["float16", "bfloat16"])
@pytest.mark.parametrize("heads", HEADS + [(6, 6, 64), (15, 3, 128), (16, 1, 256), (9, 1, 256)])
def test_chunks(pkg, heads, kind):
    """128-row tiles: rows that fill tiles exactly and not, key blocks full and not, tiles cut between CTAs, beside
    sequences of a few rows and of none."""
    lens = [64, 65, 128, 1, 200, 3000, 17, 129, 0]
    counts = [64, 33, 128, 1, 17, 300, 0, 2, 0]
    seqs = Sequences(pkg, lens, heads, seed=28)
    q, cu, host = seqs.queries(counts, getattr(torch, kind), pad=5)
    gate = torch.randn(q.shape, generator=seqs.gen, device="cuda")
    out, _, _ = attend(pkg, seqs, q, cu, counts)
    check_attention(seqs, q, host, out)
    assert (out[host[-1]:] == 77).all()
    out, _, _ = attend(pkg, seqs, q, cu, counts, gate=gate)
    check_attention(seqs, q, host, out, gate=gate)
    again, _, _ = attend(pkg, seqs, q, cu, counts, gate=gate)
    assert torch.equal(out, again)
    seqs.cache.check()


def test_chunk_values_that_grow(pkg):
    """V's groups grow by powers of ten along a sequence, each at its own pace, and logits too: what a chunk has
    summed is brought to the new power or maximum."""
    heads = (8, 1, 256)
    seqs = Sequences(pkg, [1500], heads, seed=29)
    n = seqs.lens[0]
    at = torch.arange(n, device="cuda")[:, None, None]
    pace = torch.tensor([0.0, 0.004, 0.008, -0.006], device="cuda").repeat_interleave(64)
    v = torch.randn(n, 1, 256, generator=seqs.gen, device="cuda") * 10 ** (at * pace - 3)
    k = torch.randn(n, 1, 256, generator=seqs.gen, device="cuda") * (0.02 + at / 500)
    seqs.cache.append(None, k, v, None, seqs.slots(0, 0, n), None)
    (seqs.k[0], seqs.most[0]), seqs.v[0] = quantised(k), quantised(v)[0]
    q, cu, host = seqs.queries([40], torch.bfloat16)
    out, _, _ = attend(pkg, seqs, q, cu, [40])
    ref, _, _, ds = U.attention(q, seqs.k[0], seqs.v[0], seqs.most[0], 1 / 16)
    ds = ds * (1 + 2.0 ** 12 / 256)
    for g in range(4):  # each group by its own size
        part = slice(64 * g, 64 * g + 64)
        vmax = seqs.v[0][..., part].abs().max().item()
        d = (out[..., part].double() - ref[..., part]).abs()
        assert (d <= 2.0 ** -8 * ref[..., part].abs() + (3 * 2.0 ** -11 + 2 * ds[..., None] + 2.0 ** -17) * vmax).all(), g


def test_chunk_nan_reaches_only_the_rows_that_see_it(pkg):
    """NaN keys and values inside a chunk: rows before them are untouched; a value's NaN stays in its group of dims."""
    heads = (8, 1, 128)
    seqs = Sequences(pkg, [100], heads, seed=33)
    q, cu, host = seqs.queries([60], torch.float16)
    good, _, _ = attend(pkg, seqs, q, cu, [60])
    k, v = read(seqs.cache, seqs.slots(0, 0, 100))
    bad_v = v[70:71].clone()
    bad_v[..., 64:] = math.nan
    seqs.cache.append(None, k[70:71].contiguous(), bad_v, None, seqs.slots(0, 70, 71), None)
    out, _, _ = attend(pkg, seqs, q, cu, [60])
    assert torch.equal(out[:30], good[:30]) and torch.equal(out[30:, :, :64], good[30:, :, :64])
    assert torch.isnan(out[30:, :, 64:]).all()
    seqs.cache.append(None, torch.full_like(k[:1], math.inf), v[90:91].contiguous(), None, seqs.slots(0, 90, 91), None)
    out, _, _ = attend(pkg, seqs, q, cu, [60])
    assert torch.equal(out[:30], good[:30]) and torch.equal(out[30:50, :, :64], good[30:50, :, :64])
    assert torch.isnan(out[50:]).all()


def test_chunk_queries_of_any_size(pkg):
    heads = (8, 1, 128)
    seqs = Sequences(pkg, [100], heads, seed=34)
    q, cu, host = seqs.queries([20], torch.bfloat16)
    q[0] *= 1e30
    q[1] = 0
    q[2] *= 1e-30
    out, _, _ = attend(pkg, seqs, q, cu, [20], scale=1e-6)
    assert torch.isfinite(out).all()
    ref, _, _, ds = U.attention(q, seqs.k[0], seqs.v[0], seqs.most[0], 1e-6)
    vmax, ds = seqs.v[0].abs().max(), ds * (1 + 2.0 ** 12 / 128)
    tol = 2.0 ** -8 * ref.abs() + (3 * 2.0 ** -11 + 2 * ds[..., None] + 2.0 ** -17) * vmax
    assert ((out.double() - ref).abs()[1:] <= tol[1:]).all()
    q[5, 3, 7], q[9, 0, 0] = math.nan, math.inf
    bad, _, _ = attend(pkg, seqs, q, cu, [20], scale=1e-6)
    assert torch.isnan(bad[5, 3]).all() and torch.isnan(bad[9, 0]).all()
    bad[5, 3], bad[9, 0] = out[5, 3], out[9, 0]
    assert torch.equal(bad, out)


def test_captured_and_replayed(pkg):
    """A graph of append and attention, replayed on new inputs and lengths, on a stream of its own; two graphs with
    their own workspaces in turn."""
    heads = (16, 2, 256)
    graphs = []
    for g in range(2):
        seqs = Sequences(pkg, [100, 31], heads, seed=22 + g, extra_pages=4)
        for s in range(2):  # room for the next tokens
            seqs.table[s, -(-seqs.lens[s] // 16)] = seqs.spare[s]
        q_in = torch.randn(2, 16, 256, device="cuda")
        k, v = torch.randn(2, 2, 256, device="cuda"), torch.randn(2, 2, 256, device="cuda")
        pos, slots = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.full((2,), -1, dtype=torch.int64, device="cuda")
        q = torch.empty(2, 16, 256, dtype=torch.bfloat16, device="cuda")
        out = torch.empty_like(q)
        cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
        ws = torch.empty(seqs.cache.workspace_bytes(2, 2), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            seqs.cache.append(q_in, k, v, pos, slots, q, rope_dims=64)
            seqs.cache.attention(q, cu, seqs.kv_lens, seqs.table, out, ws, 1)
        graphs.append((seqs, q_in, k, v, pos, slots, q, out, (cu, ws), graph))  # a graph's buffers live as long as it
    for step in range(3):
        for seqs, q_in, k, v, pos, slots, q, out, _, graph in graphs:
            for x in (q_in, k, v):
                x.normal_()
            pos.copy_(seqs.kv_lens)
            slots.copy_(torch.cat([seqs.slots(s, n, n + 1) for s, n in enumerate(seqs.lens)]))
            kk, most = quantised(U.normed_rotated(k, pos, rope=64))
            vv = quantised(v)[0]
            for s in range(2):
                seqs.k[s] = torch.cat([seqs.k[s], kk[s:s + 1]])
                seqs.v[s] = torch.cat([seqs.v[s], vv[s:s + 1]])
                seqs.most[s] = torch.cat([seqs.most[s], most[s:s + 1]])
                seqs.lens[s] += 1
            seqs.kv_lens.add_(1)
        torch.cuda.synchronize()
        for g in graphs:
            g[-1].replay()
        torch.cuda.synchronize()
        for seqs, q_in, k, v, pos, slots, q, out, _, graph in graphs:
            check_attention(seqs, q, [0, 1, 2], out)
            seqs.cache.check()


def test_on_another_stream(pkg):
    seqs = Sequences(pkg, [300, 40], (4, 1, 64), seed=24)
    q, cu, host = seqs.queries([1, 1], torch.float16)
    want, _, _ = attend(pkg, seqs, q, cu, [1, 1])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    out, _, _ = attend(pkg, seqs, q, cu, [1, 1], stream=side)
    side.synchronize()
    assert torch.equal(out, want)
    with torch.cuda.stream(side):
        out, _, _ = attend(pkg, seqs, q, cu, [1, 1])
    side.synchronize()
    assert torch.equal(out, want)


def test_wrapper_refusals(pkg):
    seqs = Sequences(pkg, [10], (4, 1, 64), seed=25)
    c = seqs.cache
    q, cu, _ = seqs.queries([1], torch.float16)
    ws = torch.empty(c.workspace_bytes(1, 1), dtype=torch.uint8, device="cuda")

    def call(**kw):
        a = dict(q=q, cu_seqlens=cu, kv_lens=seqs.kv_lens, block_table=seqs.table, out=torch.empty_like(q), workspace=ws,
                 max_count=1)
        a.update(kw)
        c.attention(**a)

    call()
    for kw in (dict(q=q.float()), dict(out=torch.empty_like(q).float()), dict(kv_lens=seqs.kv_lens.long()),
               dict(block_table=seqs.table[:, ::2]), dict(cu_seqlens=cu[:1]), dict(gate=q), dict(max_count=0),
               dict(workspace=ws[:8]), dict(q=q[:, :2]), dict(q=q.cpu()), dict(lse=torch.empty(1, 3, device="cuda")),
               dict(weights_in=torch.empty(1, 1, 16, device="cuda")), dict(q=q.transpose(1, 2).contiguous().transpose(1, 2))):
        with pytest.raises((ValueError, pkg.NativeError)):
            call(**kw)
    with pytest.raises(ValueError):
        pkg.Kv4Cache(torch.empty(18 * 64 + 1, dtype=torch.uint8, device="cuda"), 4, 1, 64)
    with pytest.raises(pkg.NativeError):
        pkg.Kv4Cache(seqs.pool, 33, 1, 64)
    k = torch.empty(1, 1, 64, device="cuda")
    with pytest.raises(ValueError):
        c.append(None, k, None, None, torch.zeros(1, dtype=torch.int64, device="cuda"), None)
    with pytest.raises(ValueError):
        c.append(None, k, k, None, torch.zeros(1, dtype=torch.int32, device="cuda"), None)


# ------------------------------------------------------------------ eviction

def run_evict(pkg, seqs, weights, keep, recent, with_weights=True):
    n = len(seqs.lens)
    per = -(-keep // 16)
    dst = torch.tensor(seqs.spare[:n * per], dtype=torch.int32, device="cuda").view(n, per)
    kept = torch.full((n, seqs.Hkv, keep), -9, dtype=torch.int32, device="cuda")
    lens = torch.full((n,), -9, dtype=torch.int32, device="cuda")
    wo = torch.full((n, seqs.Hkv, keep + 5), 44.0, device="cuda") if with_weights else None
    seqs.cache.evict(seqs.kv_lens, seqs.table, dst, weights, keep, recent, kept, lens, wo)
    return dst, kept, lens, wo


def check_evict(seqs, weights, keep, recent, dst, kept, lens, wo):
    got_lens, got = lens.tolist(), kept.tolist()
    for s, n in enumerate(seqs.lens):
        m = min(n, keep)
        assert got_lens[s] == m
        p = torch.arange(m, device="cuda")
        slots = dst[s, p // 16].long() * 16 + p % 16
        k, v = read(seqs.cache, slots)
        for h in range(seqs.Hkv):
            want = U.evicted(weights[s, h], n, keep, recent)
            assert got[s][h] == want + [-1] * (keep - m), (s, h)
            at = torch.tensor(want, device="cuda", dtype=torch.int64)
            assert torch.equal(k[:, h].double(), seqs.k[s][at, h]) and torch.equal(v[:, h].double(), seqs.v[s][at, h])
            if wo is not None:
                bits = lambda x: x.contiguous().view(torch.int32)  # noqa: E731
                assert torch.equal(bits(wo[s, h, :m]), bits(weights[s, h, at]))
                assert (wo[s, h, m:keep] == 0).all() and (wo[s, h, keep:] == 44).all()


@pytest.mark.parametrize("keep,recent", [(1, 0), (1, 1), (16, 4), (33, 0), (40, 40), (100, 7), (2000, 100)])
@pytest.mark.parametrize("heads", HEADS)
def test_evict(pkg, heads, keep, recent):
    lens = [1, 0, 16, 33, 34, 101, 1024, 1025, 2100]
    seqs = Sequences(pkg, lens, heads, seed=30, extra_pages=9 * (-(-keep // 16)))
    width = seqs.table.shape[1] * 16
    weights = torch.rand(len(lens), seqs.Hkv, width, generator=seqs.gen, device="cuda") ** 4
    weights[4] = 0.25  # all ties
    weights[6] = (weights[6] * 8).floor()  # many ties
    got = run_evict(pkg, seqs, weights, keep, recent)
    check_evict(seqs, weights, keep, recent, *got)
    bare = run_evict(pkg, seqs, weights, keep, recent, with_weights=False)
    assert torch.equal(bare[1], got[1])
    seqs.cache.check()


def test_evict_orders_every_float(pkg):
    """Signed zeros, infinities, NaN and negative weights by the IEEE total order."""
    seqs = Sequences(pkg, [64], (4, 1, 64), seed=31, extra_pages=8)
    values = [0.0, -0.0, math.inf, -math.inf, math.nan, -1.0, 1.0, 1e-42, -1e-42, 3e38]
    weights = torch.tensor([values[(i * 7) % 10] for i in range(seqs.table.shape[1] * 16)], device="cuda").view(1, 1, -1)
    for keep in (3, 10, 26, 40, 60):
        check_evict(seqs, weights, keep, 2, *run_evict(pkg, seqs, weights, keep, 2))


def test_evict_reports_lengths_and_pages_out_of_range(pkg):
    seqs = Sequences(pkg, [40, 40], (4, 1, 64), seed=32, extra_pages=8, pad_columns=0)
    weights = torch.rand(2, 1, 48, generator=seqs.gen, device="cuda")
    seqs.kv_lens = torch.tensor([1 << 30, -3], dtype=torch.int32, device="cuda")
    _, kept, lens, _ = run_evict(pkg, seqs, weights, 16, 0)
    assert lens.tolist() == [16, 0] and (kept[1] == -1).all() and (kept[0] < 48).all()
    with pytest.raises(pkg.NativeError, match="flag 2"):
        seqs.cache.check()
    seqs.kv_lens = torch.tensor([40, 40], dtype=torch.int32, device="cuda")
    seqs.table[0, 0] = 1 << 24
    before = seqs.pool.clone()
    run_evict(pkg, seqs, weights, 48, 0)
    with pytest.raises(pkg.NativeError, match="flag 2"):
        seqs.cache.check()
    assert before.numel() == seqs.pool.numel()


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("heads,rope", [((4, 1, 64), 16), ((16, 2, 256), 64)])
def test_prefill_decode_evict_decode(pkg, heads, rope):
    """A prompt chunk, decode steps that accumulate weights, an eviction, and decode on what is left: every output
    against the 64-bit forms over the same values."""
    Hq, Hkv, D = heads
    gen = torch.Generator(device="cuda").manual_seed(40)
    cache = new_cache(pkg, heads, 64)
    table = torch.randperm(64, generator=gen, device="cuda").int()[:60].view(2, 30).contiguous()
    n, positions, dropped = [0, 0], [0, 0], [0, 0]
    seqs = Sequences.__new__(Sequences)
    seqs.Hq, seqs.Hkv, seqs.D, seqs.cache, seqs.gen = Hq, Hkv, D, cache, gen
    seqs.table, seqs.lens = table[:, :20].contiguous(), n
    seqs.k = [torch.empty(0, Hkv, D, device="cuda", dtype=torch.float64) for _ in range(2)]
    seqs.v, seqs.most = [x.clone() for x in seqs.k], [x.clone() for x in seqs.k]
    norm = 1 + 0.1 * torch.randn(D, generator=gen, device="cuda")
    weights = torch.zeros(2, Hkv, 320, device="cuda")

    def step(counts):
        T = sum(counts)
        q_in, k, v = (torch.randn(T, h, D, generator=gen, device="cuda").bfloat16() for h in (Hq, Hkv, Hkv))
        pos = torch.cat([torch.arange(positions[s], positions[s] + c) for s, c in enumerate(counts)]).int().cuda()
        slots = torch.cat([seqs.slots(s, seqs.lens[s], seqs.lens[s] + c) for s, c in enumerate(counts)])
        q = torch.empty(T, Hq, D, dtype=torch.bfloat16, device="cuda")
        cache.append(q_in, k, v, pos, slots, q, q_norm=norm, k_norm=norm, rope_dims=rope)
        kk, most = quantised(U.normed_rotated(k, pos, norm, rope=rope))
        vv, at = quantised(v)[0], 0
        for s, c in enumerate(counts):
            seqs.k[s] = torch.cat([seqs.k[s], kk[at:at + c]])
            seqs.v[s] = torch.cat([seqs.v[s], vv[at:at + c]])
            seqs.most[s] = torch.cat([seqs.most[s], most[at:at + c]])
            seqs.lens[s] += c
            positions[s] += c
            at += c
        seqs.kv_lens = torch.tensor(seqs.lens, dtype=torch.int32, device="cuda")
        cu = torch.tensor([0, counts[0], T], dtype=torch.int32, device="cuda")
        before = weights.clone()
        out = torch.empty_like(q)
        lse = torch.empty(T, Hq, device="cuda")
        ws = torch.empty(cache.workspace_bytes(2, T), dtype=torch.uint8, device="cuda")
        cache.attention(q, cu, seqs.kv_lens, seqs.table, out, ws, max(counts), lse=lse, weights_in=weights,
                        weights_out=weights)
        check_attention(seqs, q, [0, counts[0], T], out, lse, weights, weights_in=before)

    step([150, 40])
    step([1, 60])
    for _ in range(3):
        step([1, 1])
    keep, recent = 48, 8
    kept = torch.empty(2, Hkv, keep, dtype=torch.int32, device="cuda")
    lens = torch.empty(2, dtype=torch.int32, device="cuda")
    fresh = table[:, 20:].contiguous()
    cache.evict(seqs.kv_lens, seqs.table, fresh, weights.clone(), keep, recent, kept, lens, weights)
    assert lens.tolist() == [keep, keep]
    for s in range(2):
        at = kept[s].long()  # [Hkv, keep]
        for name in ("k", "v", "most"):
            x = getattr(seqs, name)[s]
            getattr(seqs, name)[s] = torch.stack([x[at[h], h] for h in range(Hkv)], 1)
        seqs.lens[s] = keep
    seqs.table = fresh
    for counts in ([1, 1], [5, 1], [1, 20], [1, 1]):
        step(counts)
    cache.check()


# ------------------------------------------------------------------ the size of a call

def test_a_long_chunk_beside_many_decoding_sequences(pkg):
    """What bounds a call is the rows and pages that it has, not the longest chunk times the sequences: 129 decoding
    sequences and 2048 tokens of another, under a table for 262144 tokens, with statistics (8-row tiles) and without."""
    lens, counts = [1 + (i * 53) % 300 for i in range(129)] + [2100], [1] * 129 + [2048]
    seqs = Sequences(pkg, lens, (4, 2, 64), seed=41, pad_columns=(1 << 14) - 132)
    assert seqs.table.shape[1] == 1 << 14
    q, cu, host = seqs.queries(counts, torch.bfloat16)
    out, lse, weights = attend(pkg, seqs, q, cu, counts, stats=True)
    check_attention(seqs, q, host, out, lse, weights)
    del weights
    plain, _, _ = attend(pkg, seqs, q, cu, counts)
    check_attention(seqs, q, host, plain)
    seqs.cache.check()


def test_overlapping_sequences_beyond_the_bound_compute_nothing(pkg):
    """1201 sequences over the same 4096 rows, 65536 keys each: 1.2e9 places, where the rows there are allow 5e6."""
    seqs = Sequences(pkg, [16], (1, 1, 64), seed=42)
    n, T, pages = 2401, 4096, 4096
    q = torch.randn(T, 1, 64, device="cuda").half()
    cu = torch.tensor([0, T] * (n // 2 + 1), dtype=torch.int32, device="cuda")
    lens = torch.full((n,), 16 * pages, dtype=torch.int32, device="cuda")
    table = seqs.table[0, 0].expand(n, pages).contiguous()
    out, lse = torch.full_like(q, 77.0), torch.full((T, 1), 77.0, device="cuda")
    ws = torch.empty(seqs.cache.workspace_bytes(n, T), dtype=torch.uint8, device="cuda")
    seqs.cache.attention(q, cu, lens, table, out, ws, T, lse=lse)
    with pytest.raises(pkg.NativeError, match="flag 2"):
        seqs.cache.check()
    assert (out == 0).all() and (lse == -math.inf).all()


def test_evict_copies_nothing_from_a_page_that_is_not_there(pkg):
    """Keys of a source page outside the pool are skipped: their places in the destination, every page that is no
    destination, and the other sequence stay byte for byte what they were."""
    heads = (4, 2, 64)
    seqs = Sequences(pkg, [40, 40], heads, seed=43, extra_pages=8)
    page = pkg.kv4_page_bytes(2, 64)
    weights = torch.rand(2, 2, seqs.table.shape[1] * 16, generator=seqs.gen, device="cuda")
    good = seqs.pool.clone()
    dst, kept, lens, _ = run_evict(pkg, seqs, weights, 24, 4)
    check_evict(seqs, weights, 24, 4, dst, kept, lens, None)
    whole = seqs.pool.clone()
    seqs.pool.copy_(good)
    seqs.table[0, 1] = 1 << 24
    dst, again, lens, _ = run_evict(pkg, seqs, weights, 24, 4)
    with pytest.raises(pkg.NativeError, match="flag 2"):
        seqs.cache.check()
    assert torch.equal(again, kept) and lens.tolist() == [24, 24]
    now, was, full = (x.view(-1, page) for x in (seqs.pool, good, whole))
    other = torch.ones(now.shape[0], dtype=torch.bool, device="cuda")
    other[dst.flatten().long()] = False
    assert torch.equal(now[other], was[other])
    assert torch.equal(now[dst[1].long()], full[dst[1].long()])
    p = torch.arange(24, device="cuda")
    slots = dst[0, p // 16].long() * 16 + p % 16
    k, v = read(seqs.cache, slots)  # 0xFF bytes read as NaN: the places that were not written
    for h in range(2):
        gone = kept[0, h] // 16 == 1
        assert gone.any() and not gone.all()
        for got, x in ((k, seqs.k), (v, seqs.v)):
            assert torch.isnan(got[gone, h]).all()
            assert torch.equal(got[~gone, h].double(), x[0][kept[0, h].long()[~gone], h])


def test_check_waits_for_calls_on_other_streams(pkg):
    """An index out of range that a call on another stream is still to meet."""
    cache = new_cache(pkg, (2, 1, 64), 2)
    x, slots = torch.randn(1, 1, 64, device="cuda"), torch.tensor([1 << 20], device="cuda")
    a = torch.randn(8192, 8192, device="cuda")
    b = torch.mm(a, a)
    cache.append(None, x, x, None, slots % 32, None)  # kernels are loaded, which can wait for the device
    cache.check()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(10):
            torch.mm(a, a, out=b)
    cache.append(None, x, x, None, slots, None, stream=side)
    with pytest.raises(pkg.NativeError, match="flag 2"):
        cache.check()
    cache.check()  # cleared


def test_weights_and_eviction_captured_and_replayed(pkg):
    """A graph of attention that accumulates weights in place (the log-sum-exp in the workspace) and of the eviction
    that ranks by them, against the same calls made one by one, over three replays."""
    def state():
        seqs = Sequences(pkg, [100, 37, 300], (16, 2, 256), seed=44, extra_pages=12)
        q, cu, _ = seqs.queries([1, 2, 40], torch.bfloat16)
        s = dict(seqs=seqs, q=q, cu=cu, out=torch.zeros_like(q), kept=torch.full((3, 2, 60), -9, dtype=torch.int32, device="cuda"),
                 lens=torch.zeros(3, dtype=torch.int32, device="cuda"), wo=torch.zeros(3, 2, 64, device="cuda"),
                 w=torch.rand(3, 2, seqs.table.shape[1] * 16, generator=seqs.gen, device="cuda"),
                 ws=torch.empty(seqs.cache.workspace_bytes(3, 43), dtype=torch.uint8, device="cuda"),
                 dst=torch.tensor(seqs.spare[:12], dtype=torch.int32, device="cuda").view(3, 4))
        return s

    def calls(s):
        c, k = s["seqs"].cache, s["seqs"]
        c.attention(s["q"], s["cu"], k.kv_lens, k.table, s["out"], s["ws"], 40, weights_in=s["w"], weights_out=s["w"])
        c.evict(k.kv_lens, k.table, s["dst"], s["w"], 60, 8, s["kept"], s["lens"], s["wo"])

    one, two = state(), state()
    torch.cuda.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        calls(one)
    for _ in range(3):
        graph.replay()
        calls(two)
    torch.cuda.synchronize()
    for name in ("out", "kept", "lens", "wo", "w"):
        assert torch.equal(one[name], two[name]), name
    assert torch.equal(one["seqs"].pool, two["seqs"].pool)
    want = [U.evicted(two["w"][s, h], n, 60, 8) for s, n in enumerate(two["seqs"].lens) for h in range(2)]
    got = [[i for i in row if i >= 0] for row in two["kept"].view(6, 60).tolist()]
    assert got == want


def test_calls_from_two_threads(pkg):
    """Two host threads, each with its own cache, workspace and stream, give what they give one after the other."""
    import threading

    work = []
    for i, kind in enumerate((torch.float16, torch.bfloat16)):
        seqs = Sequences(pkg, [700, 64, 9], (16, 2, 256) if i else (20, 4, 128), seed=45 + i)
        counts = [60, 1, 3]
        q, cu, host = seqs.queries(counts, kind)
        want, _, _ = attend(pkg, seqs, q, cu, counts)
        work.append([seqs, q, cu, counts, want, torch.cuda.Stream(), []])
    torch.cuda.synchronize()

    def run(seqs, q, cu, counts, want, stream, got):
        with torch.cuda.stream(stream):
            for _ in range(20):
                got.append(attend(pkg, seqs, q, cu, counts)[0])

    threads = [threading.Thread(target=run, args=w) for w in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for *_, want, _, got in work:
        assert len(got) == 20 and all(torch.equal(x, want) for x in got)
