"""Host side of the 4-bit KV-cache operators, without a GPU: sizes, struct
layouts and the refusals, which come before any device work (the pointers given
here are never read)."""
import ctypes as C

import pytest

FAKE = 0x10000  # stands for device memory: refused calls do not touch it


def test_sizes(pkg):
    assert pkg.kv4_page_bytes(2, 256) == 2 * 18 * 256
    assert pkg.kv4_page_bytes(1, 64) == 18 * 64
    for bad in ((0, 64), (1, 80), (1025, 64), (-1, 128)):
        with pytest.raises(pkg.NativeError):
            pkg.kv4_page_bytes(*bad)
    assert C.sizeof(pkg.Kv4CacheDesc) == 40
    assert C.sizeof(pkg.Kv4Rows) == 24
    assert C.sizeof(pkg.Kv4AppendArgs) == 144
    assert C.sizeof(pkg.Kv4AttentionArgs) == 192
    assert C.sizeof(pkg.Kv4EvictArgs) == 104


def cache(pkg, **kw):
    d = dict(device=0, q_heads=4, kv_heads=2, head_dim=64, pages=8, pool=FAKE, status=None)
    d.update(kw)
    return pkg.Kv4CacheDesc(*[d[n] for n, _ in pkg.Kv4CacheDesc._fields_])


def refused(pkg, name, desc, args, match):
    with pytest.raises(pkg.NativeError, match=match):
        pkg._call(name, C.byref(desc) if desc is not None else None, C.byref(args), None)


@pytest.mark.parametrize("kw,match", [
    (dict(head_dim=96), "head_dim"), (dict(q_heads=5), "multiple"), (dict(q_heads=34), "16 query heads"),
    (dict(kv_heads=0), "kv_heads"), (dict(pool=None), "pool"), (dict(pool=FAKE + 8), "pool"),
    (dict(pages=0), "page count"), (dict(pages=1 << 31), "page count"), (dict(status=FAKE + 2), "status")])
def test_cache_refusals(pkg, kw, match):
    for name, args in (("append", append(pkg)), ("attention", attention(pkg)), ("evict", evict(pkg))):
        refused(pkg, "rs_qwen_kv4_" + name, cache(pkg, **kw), args, match)
    with pytest.raises(pkg.NativeError, match=match):
        pkg._call("rs_qwen_kv4_read", C.byref(cache(pkg, **kw)), 1, FAKE, 0, FAKE, FAKE, None)


def test_null_cache(pkg):
    refused(pkg, "rs_qwen_kv4_append", None, append(pkg), "null cache")
    assert pkg.load().rs_qwen_kv4_workspace_bytes(None, 1, 1) == 0
    assert pkg.load().rs_qwen_kv4_workspace_bytes(C.byref(cache(pkg, head_dim=65)), 1, 1) == 0
    assert pkg.load().rs_qwen_kv4_workspace_bytes(C.byref(cache(pkg)), 4, 4) > 0


def build(cls, d, kw):
    d.update(kw)
    return cls(*[d[n] for n, _ in cls._fields_])


def append(pkg, **kw):
    row = pkg.Kv4Rows(FAKE, 512, 64)
    return build(pkg.Kv4AppendArgs, dict(q=row, k=row, v=row, dtype=0, q_out_dtype=1, tokens=3, q_norm=FAKE, k_norm=FAKE,
                                         positions=FAKE, slots=FAKE, q_out=FAKE, epsilon=1e-6, theta=1e4, rope_dims=16,
                                         reserved=0), kw)


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=3), "dtype"), (dict(q_out_dtype=7), "dtype"), (dict(tokens=1 << 31), "too many"),
    (dict(slots=None), "slots"), (dict(slots=FAKE + 4), "slots"), (dict(q_out=FAKE + 4), "q_out"),
    (dict(q_out=None), "go together"), (dict(rope_dims=15), "rope_dims"), (dict(rope_dims=66), "rope_dims"),
    (dict(rope_dims=-2), "rope_dims"), (dict(positions=None), "positions"), (dict(theta=1.0), "theta"),
    (dict(theta=float("nan")), "theta"), (dict(epsilon=0.0), "epsilon"), (dict(epsilon=float("nan")), "epsilon"),
    (dict(q_norm=FAKE + 1), "gains")])
def test_append_refusals(pkg, kw, match):
    refused(pkg, "rs_qwen_kv4_append", cache(pkg), append(pkg, **kw), match)


def test_append_refuses_half_of_a_pair(pkg):
    none, odd = pkg.Kv4Rows(), pkg.Kv4Rows(FAKE + 1, 512, 64)
    refused(pkg, "rs_qwen_kv4_append", cache(pkg), append(pkg, v=none), "go together")
    refused(pkg, "rs_qwen_kv4_append", cache(pkg), append(pkg, q=none), "go together")
    refused(pkg, "rs_qwen_kv4_append", cache(pkg), append(pkg, q=none, k=none, v=none, q_out=None), "neither")
    refused(pkg, "rs_qwen_kv4_append", cache(pkg), append(pkg, k=odd), "aligned")


def attention(pkg, **kw):
    row = pkg.Kv4Rows(FAKE, 256, 64)
    return build(pkg.Kv4AttentionArgs, dict(q=row, gate=pkg.Kv4Rows(), out=row, dtype=1, reserved=0, n_seq=2, tokens=3,
                                            max_count=2, cu_seqlens=FAKE, kv_lens=FAKE, block_table=FAKE, table_stride=4,
                                            scale=0.0, lse=None, weights_in=None, weights_out=None, weights_stride=0,
                                            workspace=FAKE, workspace_bytes=1 << 30), kw)


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=0), "fp16 or bf16"), (dict(dtype=9), "fp16 or bf16"), (dict(tokens=1 << 29), "tokens"), (dict(n_seq=1 << 30), "sequences"),
    (dict(max_count=0), "max_count"),
    (dict(cu_seqlens=None), "cu_seqlens"), (dict(kv_lens=FAKE + 2), "kv_lens"),
    (dict(block_table=None), "block_table"), (dict(table_stride=0), "table_stride"),
    (dict(table_stride=1 << 28), "table_stride"), (dict(scale=-1.0), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(weights_in=FAKE), "weights_out"),
    (dict(weights_out=FAKE, weights_stride=0), "weights_stride"), (dict(lse=FAKE + 2), "lse"),
    (dict(n_seq=1 << 31), "too many"), (dict(tokens=1 << 31), "too many")])
def test_attention_refusals(pkg, kw, match):
    refused(pkg, "rs_qwen_kv4_attention", cache(pkg), attention(pkg, **kw), match)


def test_attention_refuses_missing_rows(pkg):
    refused(pkg, "rs_qwen_kv4_attention", cache(pkg), attention(pkg, q=pkg.Kv4Rows()), "queries or output")
    refused(pkg, "rs_qwen_kv4_attention", cache(pkg), attention(pkg, out=pkg.Kv4Rows()), "queries or output")


def evict(pkg, **kw):
    return build(pkg.Kv4EvictArgs, dict(n_seq=2, kv_lens=FAKE, src_table=FAKE, src_stride=8, dst_table=FAKE, dst_stride=2,
                                        weights=FAKE, weights_stride=128, keep=32, recent=8, kept=FAKE, new_lens=FAKE,
                                        weights_out=FAKE + 4096, weights_out_stride=32), kw)


@pytest.mark.parametrize("kw,match", [
    (dict(keep=0), "keep"), (dict(recent=-1), "recent"), (dict(recent=33), "recent"), (dict(kept=None), "missing"),
    (dict(weights=None), "missing"), (dict(new_lens=None), "missing"), (dict(src_table=FAKE + 1), "aligned"),
    (dict(src_stride=0), "src_stride"), (dict(dst_stride=1), "dst_stride"), (dict(weights_stride=0), "weights_stride"),
    (dict(weights_out_stride=31), "weights_out_stride"), (dict(weights_out=FAKE), "must not be weights"),
    (dict(n_seq=1 << 31), "too many")])
def test_evict_refusals(pkg, kw, match):
    refused(pkg, "rs_qwen_kv4_evict", cache(pkg), evict(pkg, **kw), match)


@pytest.mark.parametrize("args,match", [
    ((1, None, 0, FAKE, FAKE), "slots"), ((1, FAKE + 4, 0, FAKE, FAKE), "slots"), ((1, FAKE, 3, FAKE, FAKE), "dtype"),
    ((1, FAKE, 0, None, FAKE), "outputs"), ((1, FAKE, 0, FAKE, FAKE + 8), "outputs"), ((1 << 31, FAKE, 0, FAKE, FAKE), "many")])
def test_read_refusals(pkg, args, match):
    with pytest.raises(pkg.NativeError, match=match):
        pkg._call("rs_qwen_kv4_read", C.byref(cache(pkg)), *args, None)


def test_empty_calls_succeed_without_a_device(pkg):
    c = C.byref(cache(pkg))
    pkg._call("rs_qwen_kv4_append", c, C.byref(append(pkg, tokens=0)), None)
    pkg._call("rs_qwen_kv4_attention", c, C.byref(attention(pkg, tokens=0)), None)
    pkg._call("rs_qwen_kv4_attention", c, C.byref(attention(pkg, n_seq=0)), None)
    pkg._call("rs_qwen_kv4_evict", c, C.byref(evict(pkg, n_seq=0)), None)
    pkg._call("rs_qwen_kv4_read", c, 0, None, 0, None, None, None)


@pytest.mark.parametrize("kw", [
    # 2^20 tiles of 128 rows, each of up to 2^20 blocks of 64 keys
    dict(dtype=2, n_seq=1, tokens=1 << 26, max_count=1 << 26, table_stride=1 << 22),
    # with weights: 2^16 tiles of 8 rows over up to 2^23 page pairs, and 2^18 pieces of 64 pages for each of 2^15 sequences
    dict(n_seq=1 << 15, tokens=1 << 15, max_count=1, table_stride=1 << 24, weights_out=FAKE, weights_stride=1 << 28),
    dict(n_seq=1 << 12, tokens=1 << 26, max_count=1 << 14, table_stride=1 << 24)])
def test_attention_refuses_too_much_work_before_any_launch(pkg, kw):
    """The kernels' 32-bit places: such a call is refused on the host's values alone, with nothing enqueued."""
    refused(pkg, "rs_qwen_kv4_attention", cache(pkg), attention(pkg, **kw), "split the call")


@pytest.mark.parametrize("stats", [False, True])
def test_attention_accepts_a_long_chunk_beside_many_sequences(pkg, stats):
    """The bound counts the rows that a call has, not the longest chunk for every sequence: this one is refused for
    its missing workspace (or device) alone."""
    kw = dict(weights_out=FAKE, weights_stride=1 << 18) if stats else {}
    args = attention(pkg, dtype=2, n_seq=130, tokens=2177, max_count=2048, table_stride=1 << 14, workspace=None, **kw)
    with pytest.raises(pkg.NativeError) as e:
        pkg._call("rs_qwen_kv4_attention", C.byref(cache(pkg)), C.byref(args), None)
    assert "split the call" not in str(e.value)
