"""The 128-row tiles of the 4-bit cache's attention (bf16 rows, more than 32 per KV
head, neither log-sum-exp nor weights) where they can go wrong: values that are
not finite, pages that are not there, rows without keys, far-off magnitudes, views
of any alignment, many sequences, offsets, graphs and streams."""
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


def attend(seqs, q, cu, counts, out=None, gate=None, **kw):
    out = torch.full_like(q, 77.0) if out is None else out
    ws = torch.empty(seqs.cache.workspace_bytes(len(counts), max(1, q.shape[0])), dtype=torch.uint8, device="cuda")
    seqs.cache.attention(q, cu, seqs.kv_lens, seqs.table, out, ws, max(1, max(counts)), gate=gate, **kw)
    return out


def check_rows(seqs, s, q, out, scale=None, hidden=()):
    """Rows q, out [n, Hq, D] of sequence s, its last n tokens, against 64 bits; keys in `hidden` are not in the cache.
    Tolerance as in check_attention for these tiles: operands of 2^-11 (logits by 2^-11 of sum |q| |k|), softmax
    weights and values by 2^-11 of the largest value each, 32-bit sums, one rounding of the result. A value that is
    NaN makes its group of 64 dims NaN in the rows that see it, a key all of them."""
    n, L, G = q.shape[0], seqs.lens[s], seqs.Hq // seqs.Hkv
    scale = scale or seqs.D ** -0.5
    if not L:
        assert (out == 0).all()
        return
    k, v = seqs.k[s].repeat_interleave(G, 1), seqs.v[s].repeat_interleave(G, 1)
    bad_k, bad_v = torch.isnan(k).any(-1), torch.isnan(v)  # [L, Hq], [L, Hq, D]
    j = torch.arange(L, device="cuda")
    sees = j[None, :] <= (L - n + torch.arange(n, device="cuda"))[:, None]  # [n, L]
    for i in hidden:
        sees[:, i] = False
    x = torch.einsum("nhd,lhd->hnl", q.double(), k.nan_to_num()) * scale
    x = x.masked_fill(~sees[None], -math.inf)
    p = torch.where(sees.any(-1)[None, :, None], torch.softmax(x, -1), 0.0)
    ref = torch.einsum("hnl,lhd->nhd", p, v.nan_to_num())
    none = torch.einsum("nl,lhd->nhd", sees.double(), (bad_v | bad_k[..., None]).double()) > 0
    none |= sees.any(-1)[:, None, None] & ~torch.isfinite(q.double()).all(-1, keepdim=True)
    assert torch.equal(torch.isnan(out), none)
    most = seqs.most[s].nan_to_num().amax(0).repeat_interleave(G, 0)
    mass = torch.einsum("nhd,hd->nh", q.double().nan_to_num(0, 0, 0).abs(), most) * scale
    ds = (2.0 ** -11 + seqs.D * 2.0 ** -23) * mass
    vmax = v.nan_to_num().abs().max()
    loose = (3 * 2.0 ** -11 + 2 * ds[..., None] + 2.0 ** -18) * vmax
    tol = 2.0 ** -8 * (ref.abs() + loose) + loose
    d = (out.double() - ref).abs()
    assert (d <= tol)[~none].all(), d[~none].max()


@pytest.mark.parametrize("heads", HEADS)
def test_nan_reaches_only_the_rows_that_see_it(pkg, heads):
    """A NaN in one group of a value and an infinite key inside a chunk's own tokens."""
    Hq, Hkv, D = heads
    seqs = Sequences(pkg, [300, 170], heads, seed=50)
    counts = [200, 170]
    q, cu, host = seqs.queries(counts, torch.bfloat16)
    zero = torch.zeros(1, Hkv, D, device="cuda")
    for s, at in ((0, 150), (1, 69)):
        v = torch.randn(1, Hkv, D, generator=seqs.gen, device="cuda")
        v[:, :, D - 64:] = math.nan
        seqs.cache.append(None, zero, v, None, seqs.slots(s, at, at + 1), None)
        seqs.k[s][at], seqs.v[s][at], seqs.most[s][at] = 0, quantised(v)[0][0], 0
    out = attend(seqs, q, cu, counts)
    for s in range(2):
        check_rows(seqs, s, q[host[s]:host[s + 1]], out[host[s]:host[s + 1]])
    bad = torch.full((1, Hkv, D), math.inf, device="cuda")
    seqs.cache.append(None, bad, zero, None, seqs.slots(0, 250, 251), None)
    seqs.k[0][250], seqs.v[0][250], seqs.most[0][250] = math.nan, 0, 0
    out = attend(seqs, q, cu, counts)
    for s in range(2):
        check_rows(seqs, s, q[host[s]:host[s + 1]], out[host[s]:host[s + 1]])
    seqs.cache.check()


@pytest.mark.parametrize("value", [-3.4e38, 3.4e38])
@pytest.mark.parametrize("stats", [False, True])
def test_minimum_that_bf16_has_no_number_for(pkg, value, stats):
    """A finite 32-bit group whose minimum rounds to an infinity in bf16 is stored as NaN, so rows that do not see it
    are untouched (an infinite operand times a weight of zero would be NaN in all of them)."""
    seqs = Sequences(pkg, [170], (8, 1, 128), seed=60)
    q, cu, host = seqs.queries([170], torch.bfloat16)
    v = torch.randn(1, 1, 128, generator=seqs.gen, device="cuda")
    v[:, :, 64:] = value
    zero = torch.zeros_like(v)
    seqs.cache.append(None, zero, v, None, seqs.slots(0, 69, 70), None)
    k, got = torch.empty_like(v), torch.empty_like(v)
    seqs.cache.read(seqs.slots(0, 69, 70), k, got)
    assert torch.isnan(got[..., 64:]).all() and torch.equal(got[..., :64].double(), quantised(v)[0][..., :64])
    seqs.k[0][69], seqs.v[0][69], seqs.most[0][69] = 0, got[0].double(), 0
    lse = torch.empty(170, 8, device="cuda") if stats else None  # with it, the 8-row kernel
    out = attend(seqs, q, cu, [170], lse=lse)
    check_rows(seqs, 0, q, out)


@pytest.mark.parametrize("heads", HEADS + [(6, 6, 64)])
def test_rows_that_see_no_key(pkg, heads):
    """More query tokens than cached keys: the first ones are zero, whatever their query row holds; a row with a NaN
    or an infinity that sees a key is NaN."""
    lens, counts = [3, 0, 20, 100], [40, 36, 164, 150]
    seqs = Sequences(pkg, lens, heads, seed=51)
    q, cu, host = seqs.queries(counts, torch.bfloat16)
    out = attend(seqs, q, cu, counts)
    check_attention(seqs, q, host, out)
    for s, (n, c) in enumerate(zip(lens, counts)):
        for row, value in ((0, math.nan), (c - n - 1, math.inf), (min(c - 1, c - n + 1), math.nan), (c - 1, math.inf)):
            q[host[s] + row, row % heads[0], 5] = value
    out = attend(seqs, q, cu, counts)
    for s, (n, c) in enumerate(zip(lens, counts)):
        check_rows(seqs, s, q[host[s]:host[s + 1]], out[host[s]:host[s + 1]])
        assert (out[host[s]:host[s] + c - n] == 0).all()


@pytest.mark.parametrize("spread,scale", [(30.0, 0.0), (1.0, 8.0), (1e-4, 0.25), (3e4, 1e-6), (1e4, 1e4)])
@pytest.mark.parametrize("heads", HEADS)
def test_large_and_small_logits(pkg, heads, spread, scale):
    """Up to maxima beyond 2^24, where the products are rounded before they are subtracted."""
    seqs = Sequences(pkg, [40, 700], heads, seed=52, spread=spread)
    q, cu, host = seqs.queries([40, 70], torch.bfloat16)
    out = attend(seqs, q, cu, [40, 70], scale=scale)
    check_attention(seqs, q, host, out, scale=scale)


@pytest.mark.parametrize("key,query", [(1e-36, 1e36), (1e-37, 1e37), (1e-38, 3e37), (1e36, 1e-36), (1e-30, 1.0), (3e37, 1e-37), (3e37, 1e-38)])
def test_products_of_far_magnitudes(pkg, key, query):
    """Keys and queries at opposite ends of the range: their product is an ordinary logit."""
    heads = (8, 1, 128)
    seqs = Sequences(pkg, [200], heads, seed=53, spread=key)
    q, cu, host = seqs.queries([60], torch.float32)
    q = (q * query).to(torch.bfloat16)
    out = attend(seqs, q, cu, [60])
    check_rows(seqs, 0, q, out)


@pytest.mark.parametrize("heads", HEADS)
def test_pages_out_of_range_count_as_absent(pkg, heads):
    lens, counts = [40, 300, 33], [36, 290, 33]
    seqs = Sequences(pkg, lens, heads, seed=54)
    q, cu, host = seqs.queries(counts, torch.bfloat16)
    gone = [[(0, 1 << 20)], [(1, -7), (4, 1 << 24), (5, -1), (6, -1), (7, -1), (18, 1 << 30)], [(0, -1), (1, -1), (2, -1)]]
    for s, pages in enumerate(gone):
        for page, value in pages:
            seqs.table[s, page] = value
    out = attend(seqs, q, cu, counts)
    with pytest.raises(pkg.NativeError, match="flag 2"):
        seqs.cache.check()
    for s, pages in enumerate(gone):
        hidden = [i for page, _ in pages for i in range(16 * page, min(lens[s], 16 * page + 16))]
        check_rows(seqs, s, q[host[s]:host[s + 1]], out[host[s]:host[s + 1]], hidden=hidden)
    assert (out[host[2]:host[3]] == 0).all()


def test_strided_queries_gates_and_outputs(pkg):
    """Views of any start and stride give the bits of contiguous rows."""
    heads = (8, 2, 128)
    seqs = Sequences(pkg, [150, 7, 400], heads, seed=55)
    counts = [150, 5, 100]
    q, cu, host = seqs.queries(counts, torch.bfloat16)
    T = q.shape[0]
    gate = torch.randn(T, 8, 128, generator=seqs.gen, device="cuda")
    want = attend(seqs, q, cu, counts, gate=gate)
    check_attention(seqs, q, host, want, gate=gate)
    for lead, tail in ((0, 0), (1, 2), (8, 8), (2, 5)):
        buf = torch.zeros(T, 8 * 2 * 128 + lead + tail, dtype=torch.bfloat16, device="cuda")
        view = buf[:, lead:lead + 2048].unflatten(1, (8, 2, 128))[:, :, 1]
        view.copy_(q)
        gates = torch.zeros(T, 8, 128 + lead, device="cuda")
        gates[:, :, lead:] = gate
        outs = torch.full((8, T, 128 + lead), 3.0, dtype=torch.bfloat16, device="cuda")
        attend(seqs, view, cu, counts, out=outs[:, :, lead:].transpose(0, 1), gate=gates[:, :, lead:])
        assert torch.equal(outs[:, :, lead:].transpose(0, 1), want)
        assert (outs[:, :, :lead] == 3).all()


def test_many_sequences(pkg):
    """More sequences than the kernels keep apart in their tables (512): long, short and empty ones in turn."""
    lens = [(i * 37) % 190 for i in range(1100)]
    counts = [min(n, (40, 1, 0, 9, 3)[i % 5]) for i, n in enumerate(lens)]
    seqs = Sequences(pkg, lens, (4, 1, 64), seed=56)
    q, cu, host = seqs.queries(counts, torch.bfloat16, pad=2)
    out = attend(seqs, q, cu, counts)
    check_attention(seqs, q, host, out)
    assert (out[host[-1]:] == 77).all()
    seqs.cache.check()


@pytest.mark.parametrize("kind", ["float16", "bfloat16"])
def test_sequences_that_start_behind_the_first_row(pkg, kind):
    """cu_seqlens[0] > 0: the rows before it are not written (128-row tiles in bf16, 8-row tiles in fp16)."""
    lens, counts = [130, 3, 64], [50, 1, 64]
    seqs = Sequences(pkg, lens, (8, 1, 128), seed=57)
    q, cu, host = seqs.queries(counts, getattr(torch, kind), pad=9)
    cu, host = cu + 7, [h + 7 for h in host]
    out = attend(seqs, q, cu, counts)
    check_attention(seqs, q, host, out)
    assert (out[:7] == 77).all() and (out[host[-1]:] == 77).all()
    seqs.cache.check()


def test_captured_and_replayed_on_two_streams(pkg):
    """Graphs of a chunk and decoding sequences, each with its own workspace, replayed side by side on their streams
    and on lengths that change between replays."""
    graphs = []
    for g in range(2):
        seqs = Sequences(pkg, [700, 90, 300], (16, 2, 256), seed=58 + g)
        counts = [260, 1, 130]
        q, cu, host = seqs.queries(counts, torch.bfloat16)
        out = torch.empty_like(q)
        ws = torch.empty(seqs.cache.workspace_bytes(3, q.shape[0]), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            seqs.cache.attention(q, cu, seqs.kv_lens, seqs.table, out, ws, 260)
        graphs.append((seqs, q, host, out, (cu, ws), side, graph))
    full = [list(g[0].lens) for g in graphs]
    for cut in (0, 5, 33):  # shorter contexts of the same pages
        for (seqs, q, *_), lens in zip(graphs, full):
            seqs.lens = [n - cut for n in lens]
            seqs.kv_lens.copy_(torch.tensor(seqs.lens, dtype=torch.int32))
            q.normal_()
        torch.cuda.synchronize()
        for seqs, q, host, out, _, side, graph in graphs:
            with torch.cuda.stream(side):
                for _ in range(5):
                    graph.replay()
        torch.cuda.synchronize()
        for (seqs, q, host, out, *_), lens in zip(graphs, full):
            part = Sequences.__new__(Sequences)
            part.__dict__.update(seqs.__dict__)
            for name in ("k", "v", "most"):
                setattr(part, name, [x[:n] for x, n in zip(getattr(seqs, name), seqs.lens)])
            check_attention(part, q, host, out)
            seqs.cache.check()
