"""The append of the 4-bit cache for steps of more than 592 tokens, whose CTAs take
several tokens and whose warps take two query rows."""
import pytest

from conftest import has_cuda

pytestmark = pytest.mark.gpu

if has_cuda():
    import torch

    import kv4_util as U
    from kv4_util import quantised


@pytest.fixture(autouse=True)
def _cuda():
    if not has_cuda():
        pytest.skip("no CUDA device")


# 592 is the last count with a token per CTA; 2, 3 and 8 tokens per CTA, with a CTA that is not full
@pytest.mark.parametrize("T", [592, 593, 1191, 4737])
@pytest.mark.parametrize("kind,fused", [("float32", True), ("bfloat16", True), ("float16", False)])
@pytest.mark.parametrize("heads,rope", [((5, 5, 64), 16), ((15, 3, 128), 128), ((16, 2, 256), 64), ((3, 1, 128), 2), ((1, 1, 256), 0)])
def test_long_appends(pkg, heads, rope, kind, fused, T):
    """Queries, keys and values against 64 bits, and the pages bit for bit against appends of at most 40 tokens."""
    Hq, Hkv, D = heads
    gen = torch.Generator(device="cuda").manual_seed(T + rope)
    dtype, pages = getattr(torch, kind), -(-T // 16) + 3
    if fused:  # views of one projection row [query, gate] x Hq, keys, values
        row = torch.randn(T, (2 * Hq + 2 * Hkv) * D, generator=gen, device="cuda").to(dtype)
        q = row[:, :2 * Hq * D].unflatten(1, (Hq, 2, D))[:, :, 0]
        k, v = (row[:, (2 * Hq + i * Hkv) * D:(2 * Hq + (i + 1) * Hkv) * D].unflatten(1, (Hkv, D)) for i in range(2))
    else:
        q, k, v = (torch.randn(T, h, D, generator=gen, device="cuda").to(dtype) for h in (Hq, Hkv, Hkv))
    pos = torch.randint(0, 200000, (T,), generator=gen, device="cuda", dtype=torch.int32)
    slots = torch.randperm(pages * 16, generator=gen, device="cuda")[:T].contiguous()
    slots[::97] = -1  # not stored; their query rows are written all the same
    qn, kn = (1 + 0.2 * torch.randn(D, generator=gen, device="cuda") for _ in range(2))
    pools = [torch.full((pages * pkg.kv4_page_bytes(Hkv, D),), 255, dtype=torch.uint8, device="cuda") for _ in range(2)]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    whole, parts = (pkg.Kv4Cache(p, Hq, Hkv, D, status=status) for p in pools)
    out = torch.empty(T, Hq, D, dtype=torch.bfloat16 if kind == "float32" else dtype, device="cuda")
    again = torch.empty_like(out)
    opts = dict(q_norm=qn, k_norm=kn, epsilon=1e-6, theta=1e6, rope_dims=rope)
    whole.append(q, k, v, pos, slots, out, **opts)
    for a in range(0, T, 40):
        z = min(T, a + 40)
        parts.append(q[a:z], k[a:z], v[a:z], pos[a:z], slots[a:z], again[a:z], **opts)
    assert torch.equal(pools[0], pools[1]) and torch.equal(out, again)
    want = U.normed_rotated(q, pos, qn, 1e-6, 1e6, rope)
    # as for the short appends: a sum of D squares, halved by the root, and a dozen roundings in 32 bits, a rotated
    # value with its partner's error; then one rounding to the output's type
    size = want.abs() + (want.abs().amax(-1, keepdim=True) if rope else 0)
    tiny = torch.finfo(out.dtype).tiny * torch.finfo(out.dtype).eps
    tol = torch.finfo(out.dtype).eps / 2 * want.abs() + (D / 2 + 12) * 2.0 ** -24 * size + tiny
    assert ((out.double() - want).abs() <= tol * (1 + 2.0 ** -8)).all()
    got_k, got_v = (torch.empty(T, Hkv, D, device="cuda") for _ in range(2))
    whole.read(slots, got_k, got_v)
    there = slots >= 0
    for got, x in ((got_k, U.normed_rotated(k, pos, kn, 1e-6, 1e6, rope)), (got_v, v)):
        assert torch.equal(got[there].double(), quantised(x)[0][there]) and not got[~there].any()
    whole.check()
