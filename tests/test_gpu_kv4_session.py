"""Sessions on 4-bit attention pages (rs_qwen_device_kv4): the cache that steps
leave, logits against the FP64 oracle run on the values read back, forks,
verify, synthetic states, accumulated attention weights and eviction.

The tiny decoder has one attention layer behind its DeltaNet layers, so its keys
and values depend on the tokens alone and are compared bit for bit between runs.
"""
import ctypes as C

import numpy as np
import pytest
import torch

from conftest import has_cuda
from kv4_util import evicted, quantised

SEED, CONTEXT = 77, 512
HEADS, KV_HEADS, DIM, ROPE, THETA = 4, 2, 64, 16, 1e7
G = HEADS // KV_HEADS
PER = KV_HEADS * CONTEXT * DIM  # K (or V) floats of the attention layer at the end of a snapshot


def tiny(mod, context=CONTEXT):
    return mod.config(hidden=256, layers=4, vocab=4096, q_heads=HEADS, kv_heads=KV_HEADS, head_dim=DIM, key_heads=2,
                      value_heads=4, key_dim=64, value_dim=64, experts=16, top=2, intermediate=128, shared=128,
                      context=context, rope_dims=ROPE, theta=THETA)


@pytest.fixture(scope="module")
def store(pkg):
    if not has_cuda():
        pytest.skip("no CUDA device")
    store = pkg.WeightStore().synthetic(tiny(pkg), SEED, mtp=True)
    yield store
    store.close()


@pytest.fixture
def make(pkg, store):
    made = []

    def session(kv4=True, track=False, context=CONTEXT, slots=24):
        s = pkg.DeviceSession(store, tiny(pkg, context), slots, 1 << 28)
        made.append(s)
        if kv4:
            s.kv4(track)
        return s

    yield session
    for s in made:
        s.close()


def prompt(n, seed=5):
    return np.random.default_rng(seed).integers(0, 4096, size=n).astype(np.uint32)


def rel_l2(a, b):
    return float(np.linalg.norm(np.float64(a) - np.float64(b)) / np.linalg.norm(np.float64(b)))


def snapshot_kv(state):
    return state[-2 * PER:].reshape(2, KV_HEADS, CONTEXT, DIM)


def test_null_handles_are_refused(pkg):
    lib, e, n = pkg.load(), C.create_string_buffer(256), C.c_size_t()
    assert lib.rs_qwen_device_kv4(None, 0, e, 256) == -1 and e.value
    assert lib.rs_qwen_device_kv4_read(None, None, 0, None, None, None, 0, C.byref(n), e, 256) == -1 and e.value
    assert lib.rs_qwen_device_kv4_evict(None, 1, None, 8, 0, None, e, 256) == -1 and e.value


@pytest.mark.gpu
@pytest.mark.parametrize("counts", [[1], [37], [5, 48, 16, 1]])
def test_cache_of_a_prefill(pkg, make, counts):
    """Against the bf16 session: the same DeltaNet state, keys and values within a 4-bit step."""
    toks = prompt(sum(counts))
    got = []
    for kv4 in (False, True):
        s = make(kv4)
        outs, _, _ = s.step_ragged([None] * len(counts), [0] * len(counts), counts, toks)
        got.append([s.snapshot(o) for o in outs])
    for ref, out, n in zip(*got, counts):
        assert np.array_equal(ref[:-2 * PER], out[:-2 * PER])
        a, b = snapshot_kv(ref).astype(np.float64), snapshot_kv(out).astype(np.float64)
        assert not b[:, :, n:].any()
        a, b = a[:, :, :n], b[:, :, :n]
        low, high = a.min(-1, keepdims=True), a.max(-1, keepdims=True)  # one group of 64 dims
        # half a step of (max - min) / 15; scale, bias and the bf16 reference's own values are within 2^-8 (so
        # 15 steps and their end points are), the two norms within 2^-20
        most = np.maximum(abs(low), abs(high))
        tol = (high - low) / 30 * (1 + 2.0 ** -7) + 2.0 ** -8 * ((high - low) + 3 * most) + 2.0 ** -20 * most
        assert (abs(a - b) <= tol).all()


@pytest.mark.gpu
def test_synthetic_state_is_the_quantised_bf16_one(pkg, make):
    n, ctx = 3001, 4096
    states = []
    for kv4 in (False, True):
        s = make(kv4, context=ctx, slots=2)
        states.append(s.snapshot(s.synthetic_state(n, 9)))
    per = KV_HEADS * ctx * DIM
    assert np.array_equal(states[0][:-2 * per], states[1][:-2 * per])
    a, b = (x[-2 * per:].reshape(2 * KV_HEADS, ctx, DIM) for x in states)
    want, _ = quantised(torch.from_numpy(a[:, :n].copy()))
    assert np.array_equal(b[:, :n], want.float().numpy()) and not b[:, n:].any()


def check_rows(pkg, sess, model, parent, start, old_state, held_kv, tokens, shift=0):
    """Feeds `tokens` behind `parent` (cache length `start`, `shift` keys evicted); every row's logits against the
    oracle on the cache as read back. held_kv(child) gives K, V [kv][start + n][d] with K at unshifted positions.
    Returns the child."""
    n = len(tokens)
    sess.set_capture(True)
    (child,), _, logits = sess.step_ragged([parent], [start + shift], [n], tokens,
                                           flags=pkg.RAGGED_LOGITS | pkg.RAGGED_ALL_ROWS)
    route = sess.debug_routing(n)
    held = np.stack(held_kv(child))
    state = np.zeros(old_state.size, np.float32)
    state[:-2 * PER] = old_state[:-2 * PER]
    snapshot_kv(state)[:, :, :start] = held[:, :, :start]
    lg, _, _, _ = model.forward(tokens, start, old_state=state, forced_routing=route, cached_kv=held[None, :, :, start:])
    for j in range(n):
        assert rel_l2(logits[j], lg[j]) <= 1e-2, j  # the tolerance of the bf16 sessions
    return child


@pytest.mark.gpu
@pytest.mark.parametrize("block", [1, 6, 40], ids=["decode", "rows", "chunk"])
@pytest.mark.parametrize("track", [False, True])
def test_steps_against_the_oracle(pkg, O, make, block, track):
    O.set_routing_slack(5e-2)
    s, model = make(track=track), O.Model(tiny(O), SEED)
    toks = prompt(150 + 2 * block)
    empty = np.zeros(pkg.state_count(tiny(pkg)), np.float32)
    cur, pos = check_rows(pkg, s, model, None, 0, empty, lambda c: s.kv4_read(c, 0)[:2], toks[:150]), 150
    for _ in range(2):
        state = s.snapshot(cur)
        cur = check_rows(pkg, s, model, cur, pos, state, lambda c: s.kv4_read(c, 0)[:2], toks[pos:pos + block])
        pos += block
    kv = snapshot_kv(s.snapshot(cur))
    k, v, _ = s.kv4_read(cur, 0)
    assert np.array_equal(kv[0, :, :pos], k) and np.array_equal(kv[1, :, :pos], v)


@pytest.mark.gpu
@pytest.mark.parametrize("track", [False, True])
def test_wide_heads_against_the_oracle(pkg, O, track):
    """16 query heads and 2 KV heads of 256: a prefill, a block of 40 tokens (128-row tiles without tracking) and
    single tokens."""
    if not has_cuda():
        pytest.skip("no CUDA device")
    O.set_routing_slack(5e-2)
    cfg = pkg.config1(layers=4, context=256)
    store = pkg.WeightStore().synthetic(cfg, SEED)
    s = pkg.DeviceSession(store, cfg, slots=4, budget_bytes=1 << 28).kv4(track)
    model = O.Model(O.config1(layers=4, context=256), SEED)
    try:
        s.set_capture(True)
        toks = np.random.default_rng(3).integers(0, cfg.vocab, size=72).astype(np.uint32)
        cur, state, pos = None, None, 0
        for n in (30, 40, 1, 1):
            (cur,), _, logits = s.step_ragged([cur], [pos], [n], toks[pos:pos + n],
                                              flags=pkg.RAGGED_LOGITS | pkg.RAGGED_ALL_ROWS)
            route = s.debug_routing(n)
            held = np.stack(s.kv4_read(cur, 0)[:2])[None, :, :, pos:]
            lg, _, _, _ = model.forward(toks[pos:pos + n], pos, old_state=state, forced_routing=route, cached_kv=held)
            assert max(rel_l2(logits[j], lg[j]) for j in range(n)) <= 1e-2
            state, pos = s.snapshot(cur), pos + n
        s.release(cur)
    finally:
        s.close()
        store.close()


@pytest.mark.gpu
def test_forks_copy_the_shared_page(pkg, make):
    s = make()
    toks = prompt(21)

    def chain(consume_flag, tails):
        (cur,), _, _ = s.step_ragged([None], [0], [21], toks)
        out = []
        for t in tails:
            (c,), _, _ = s.step_ragged([cur], [21], [len(t)], t, flags=pkg.RAGGED_SAMPLED | consume_flag)
            out.append(c)
        return cur, out

    tails = [prompt(3, 1), prompt(18, 2), prompt(1, 3)]
    parent, kids = chain(0, tails)
    before = s.snapshot(parent)
    for t, kid in zip(tails, kids):
        _, (alone,) = chain(pkg.RAGGED_CONSUME, [t])
        assert np.array_equal(s.snapshot(kid), s.snapshot(alone))
    assert np.array_equal(s.snapshot(parent), before)


@pytest.mark.gpu
def test_verify_accept(pkg, make):
    s = make()
    lens = [5, 31, 16]
    outs, seeds, _ = s.step_ragged([None] * 3, [0] * 3, lens, prompt(sum(lens)))
    chains, rows = [], []
    for o, n, t in zip(outs, lens, seeds):
        ids, got, cur, tok = [], [], o, int(t)
        for j in range(4):
            (cur,), x, _ = s.step_ragged([cur], [n + j], [1], [tok])
            tok = int(x[0])
            ids.append(cur)
            got.append(tok)
        chains.append(ids)
        rows.append(got)
    drafts = [rows[0][:3], [(rows[1][0] + 1) % 4096], rows[2][:1] + [(rows[2][1] + 1) % 4096]]
    made, accepted, emitted = s.verify_accept(outs, [int(x) for x in seeds], drafts)
    assert list(accepted) == [3, 0, 1]
    for i, a in enumerate(accepted):
        assert emitted[i] == rows[i][:a + 1]
        assert np.array_equal(s.snapshot(made[i]), s.snapshot(chains[i][a]))


@pytest.mark.gpu
def test_draft_head_beside_4_bit_pages(pkg, O, make, store):
    """The MTP head drafts from hidden rows of a 4-bit session, on bf16 pages of its own."""
    O.set_routing_slack(5e-2)
    s, model = make(), O.Model(tiny(O), SEED, mtp=True)
    s.mtp_attach(store)
    n = 6
    (target,), _, _ = s.step_ragged([None], [0], [n], prompt(n), flags=pkg.RAGGED_SAMPLED | pkg.RAGGED_HIDDEN)
    before = s.snapshot(target)
    s.set_capture(True)
    draft, logits = s.mtp_step(None, target, prompt(n, 6))
    kv = np.zeros(2 * PER, np.float64)
    want, hidden = model.mtp_forward(prompt(n, 6), 0, s.hidden_snapshot(target, n).astype(np.float64), kv,
                                     forced_routing=s.debug_routing(n)[0])
    assert rel_l2(logits, want[-1]) <= 1e-2
    k, v, rows = s.mtp_snapshot(draft, n)
    kv = kv.reshape(2, KV_HEADS, CONTEXT, DIM)
    assert rel_l2(rows, hidden) <= 1e-2 and rel_l2(k[:, :n], kv[0, :, :n]) <= 1e-2 and rel_l2(v[:, :n], kv[1, :, :n]) <= 1e-2
    assert np.array_equal(s.snapshot(target), before)
    s.mtp_release(draft)
    s.release(target)


def rotated(k, by):
    """Keys [.., d] moved `by` positions along the rotation (64 bits)."""
    j = np.arange(ROPE // 2)
    angle = by * np.float64(np.float32(THETA)) ** (-2 * j / ROPE)
    a, b, out = np.float64(k[..., :ROPE // 2]), np.float64(k[..., ROPE // 2:ROPE]), np.float64(k)
    out[..., :ROPE // 2] = a * np.cos(angle) - b * np.sin(angle)
    out[..., ROPE // 2:ROPE] = a * np.sin(angle) + b * np.cos(angle)
    return out


# Every query row adds 1 to a KV head's weights. A logit's 32-bit sum over 64 products is off by 64 x 2^-23 of its
# products' magnitudes, at most 9 (|q| = 8, |k| <= 9, scale 1/8), in the weight and in the row's sum; the two
# exponentials by 2^-21 each.
WEIGHT_TOL = 2 * (64 * 2.0 ** -23 * 9 + 2.0 ** -21)


@pytest.mark.gpu
def test_eviction_against_the_oracle(pkg, O, make):
    O.set_routing_slack(5e-2)
    s, model = make(track=True), O.Model(tiny(O), SEED)
    lens = [190, 37]
    toks = prompt(sum(lens))
    ids, _, _ = s.step_ragged([None] * 2, [0] * 2, lens, toks)
    for i, n in enumerate(lens):
        w = s.kv4_read(ids[i], 0, weights=True)[2]
        assert (w >= 0).all() and (abs(w.sum(1, dtype=np.float64) - G * n) <= WEIGHT_TOL * G * n).all()
    fed = list(lens)
    for keep, recent in [(130, 8), (113, 113), (512, 3)]:
        before = [s.kv4_read(x, 0, weights=True) for x in ids]
        state = [None] * 2
        made = s.kv4_evict(ids, keep, recent)
        for i in range(2):
            k, v, w = before[i]
            k2, v2, w2 = s.kv4_read(made[i], 0, weights=True)
            left = min(keep, k.shape[1])
            assert k2.shape[1] == left and made[i].position == fed[i]
            for h in range(KV_HEADS):
                stay = evicted(torch.from_numpy(w[h]), k.shape[1], keep, recent)
                assert np.array_equal(k2[h], k[h, stay]) and np.array_equal(v2[h], v[h, stay])
                assert np.array_equal(w2[h], w[h, stay])
            # the version that lost keys is as it was
            assert all(np.array_equal(x, y) for x, y in zip(before[i], s.kv4_read(ids[i], 0, weights=True)))
        if made[0].position != s.kv4_read(made[0], 0)[0].shape[1]:
            with pytest.raises(pkg.NativeError, match="evicted"):
                s.snapshot(made[0])
        # three tokens of the longer sequence on what is left, its keys moved back to their places in the cache
        held = s.kv4_read(made[0], 0)[0].shape[1]
        shift = fed[0] - held
        gdn = deltanet(pkg, make, toks, fed[0], lens)
        state = np.concatenate([gdn, np.zeros(2 * PER, np.float32)])

        def held_kv(c):
            k, v, _ = s.kv4_read(c, 0)
            return rotated(k, -shift), v

        child = check_rows(pkg, s, model, made[0], held, state, held_kv, prompt(3, fed[0]), shift)
        toks = np.concatenate([toks[:fed[0]], prompt(3, fed[0]), toks[fed[0]:]])
        k2, _, w2 = s.kv4_read(made[0], 0, weights=True)
        k3, _, w3 = s.kv4_read(child, 0, weights=True)
        assert np.array_equal(k3[:, :held], k2)
        rise = w3.sum(1, dtype=np.float64) - w2.sum(1, dtype=np.float64)
        # beside the rows' own weight, each key's sum is rounded to 32 bits
        assert (abs(rise - 3 * G) <= WEIGHT_TOL * 3 * G + 2.0 ** -24 * w3.sum(1)).all()
        for x in ids:
            s.release(x)
        s.release(made[0])
        ids, fed[0] = [child, made[1]], fed[0] + 3
    assert s.drain() == 2


def deltanet(pkg, make, toks, n, lens):
    """DeltaNet part of the state after the first n tokens, fed as the test feeds them: lens[0] at once, then
    threes. Attention comes behind every DeltaNet layer, so the cache does not matter."""
    s = make(False)
    (cur,), _, _ = s.step_ragged([None], [0], [lens[0]], toks[:lens[0]])
    for at in range(lens[0], n, 3):
        (cur,), _, _ = s.step_ragged([cur], [at], [3], toks[at:at + 3], flags=pkg.RAGGED_SAMPLED | pkg.RAGGED_CONSUME)
    return s.snapshot(cur)[:-2 * PER]


@pytest.mark.gpu
def test_keeping_everything_changes_nothing(pkg, make):
    s = make(track=True)
    (a,), _, _ = s.step_ragged([None], [0], [75], prompt(75))
    (b,) = s.kv4_evict([a], 75, 0)
    assert np.array_equal(s.snapshot(a), s.snapshot(b))
    for t in prompt(3, 8):
        (a,), _, x = s.step_ragged([a], [a.position], [1], [t], flags=pkg.RAGGED_LOGITS)
        (b,), _, y = s.step_ragged([b], [b.position], [1], [t], flags=pkg.RAGGED_LOGITS | pkg.RAGGED_CONSUME)
        assert np.array_equal(x, y)
        assert all(np.array_equal(p, q) for p, q in zip(s.kv4_read(a, 0, True), s.kv4_read(b, 0, True)))


@pytest.mark.gpu
def test_evicted_versions_fork_and_free_their_pages(pkg, make):
    s = make(track=True, slots=6)
    for _ in range(40):  # more pages in all than the context's
        (a,), _, _ = s.step_ragged([None], [0], [100], prompt(100))
        b, c = s.kv4_evict([a, a], 37, 5)  # the same version twice
        kids = [s.step_ragged([b], [100], [len(t)], t)[0][0] for t in (prompt(2, 1), prompt(14, 2))]
        held = s.kv4_read(b, 0)
        for kid, n in zip(kids, (2, 14)):
            k, v, _ = s.kv4_read(kid, 0)
            assert k.shape[1] == 37 + n
            assert np.array_equal(k[:, :37], held[0]) and np.array_equal(v[:, :37], held[1])
        assert all(np.array_equal(x, y) for x, y in zip(held[:2], s.kv4_read(c, 0)[:2]))
        for x in (a, b, c, *kids):
            s.release(x)
    assert s.drain() == 0


@pytest.mark.gpu
def test_refusals(pkg, make, store):
    plain = make(False)
    (a,), _, _ = plain.step_ragged([None], [0], [3], prompt(3))
    with pytest.raises(pkg.NativeError, match="precede admission"):
        plain.kv4()
    with pytest.raises(pkg.NativeError, match="not 4-bit"):
        plain.kv4_read(a, 0)
    with pytest.raises(pkg.NativeError, match="tracked weights"):
        plain.kv4_evict([a], 2, 0)
    drafting = make(False)
    drafting.mtp_attach(store)
    with pytest.raises(pkg.NativeError, match="MTP"):
        drafting.kv4()
    s = make()
    with pytest.raises(pkg.NativeError, match="already"):
        s.kv4()
    (a,), _, _ = s.step_ragged([None], [0], [3], prompt(3))
    with pytest.raises(pkg.NativeError, match="tracked weights"):
        s.kv4_evict([a], 2, 0)
    with pytest.raises(pkg.NativeError, match="does not track"):
        s.kv4_read(a, 0, weights=True)
    with pytest.raises(pkg.NativeError, match="layer out of range"):
        s.kv4_read(a, 1)
    t = make(track=True, slots=3)
    (a,), _, _ = t.step_ragged([None], [0], [3], prompt(3))
    for keep, recent in ((0, 0), (2, 3), (CONTEXT + 1, 0)):
        with pytest.raises(pkg.NativeError, match="keep"):
            t.kv4_evict([a], keep, recent)
    with pytest.raises(pkg.NativeError, match="batch"):
        t.kv4_evict([], 2, 0)
    with pytest.raises(pkg.NativeError, match="tracks"):
        t.verify_accept([a], [1], [[2]])
    with pytest.raises(pkg.NativeError, match="budget"):
        t.kv4_evict([a, a, a], 2, 0)
    t.release(a)
    with pytest.raises(pkg.NativeError):
        t.kv4_evict([a], 2, 0)
    assert t.drain() == 0


@pytest.mark.gpu
def test_more_pages_in_the_same_budget(pkg, make):
    """A budget that holds 2 contexts in bf16 holds 7 in 4 bits."""
    s = make()
    assert s.synthetic_state(CONTEXT, 1).position == CONTEXT
    cfg = tiny(pkg)
    gdn = 3 * ((4 * 64 * 64) + (3 * (2 * 2 * 64 + 4 * 64))) * 4  # state and conv history of the DeltaNet layers
    budget = 8 * gdn + 2 * CONTEXT * 2 * KV_HEADS * DIM * 2 + 4096
    for kv4, most in ((False, 2), (True, 7)):
        sess = pkg.DeviceSession(s.store, cfg, 8, budget)
        if kv4:
            sess.kv4()
        for i in range(most):
            sess.synthetic_state(CONTEXT, i)
        with pytest.raises(pkg.NativeError, match="budget|exhausted"):
            sess.synthetic_state(CONTEXT, 9)
        sess.close()


@pytest.mark.gpu
def test_a_long_prompt_beside_many_decoding_sequences(pkg, store):
    """A tracked session with room for 262144 tokens: 129 sequences decode while one feeds 2048 tokens. Caches are
    those of the same tokens fed apart, to a 4-bit step, and every row gives a weight of one to each KV head's keys."""
    n, ctx, long = 129, 1 << 18, 2048
    s = pkg.DeviceSession(store, tiny(pkg, ctx), 2 * n + 4, 3 << 30).kv4(track=True)
    parents, _, _ = s.step_ragged([None] * n, [0] * n, [5] * n, prompt(5 * n, 11))
    tails, text = prompt(n, 12), prompt(long, 13)
    alone = []
    for i in (0, 64, n - 1):
        (c,), _, _ = s.step_ragged([parents[i]], [5], [1], tails[i:i + 1])
        alone.append((i, s.kv4_read(c, 0)))
        s.release(c)
    (c,), _, _ = s.step_ragged([None], [0], [long], text)
    alone.append((n, s.kv4_read(c, 0)))
    s.release(c)
    kids, _, _ = s.step_ragged(parents + [None], [5] * n + [0], [1] * n + [long], np.concatenate([tails, text]),
                               flags=pkg.RAGGED_SAMPLED | pkg.RAGGED_CONSUME)
    for i, held in alone:
        fed = long if i == n else 6
        k, v, w = s.kv4_read(kids[i], 0, weights=True)
        for a, b in zip(held[:2], (k, v)):
            a, b = np.float64(a), np.float64(b)
            assert a.shape == b.shape == (KV_HEADS, fed, DIM)
            # projections of another batch size may be summed in another order: a nibble moves by one at most, scale
            # and bias by a bf16 step (2^-7 of themselves)
            low, high = a.min(-1, keepdims=True), a.max(-1, keepdims=True)
            tol = (high - low) * (1 / 15 + 2.0 ** -7) + 2.0 ** -7 * np.maximum(abs(low), abs(high))
            assert (abs(a - b) <= tol).all()
        # beside the rows' own weight, each key's sum of at most G * fed terms is rounded to 32 bits
        assert (abs(w.sum(1, dtype=np.float64) - G * fed) <= (WEIGHT_TOL + G * fed * 2.0 ** -24) * G * fed).all()
    assert s.drain() == n + 1
    s.close()


@pytest.mark.gpu
def test_a_step_that_is_too_large_keeps_its_parents(pkg, store):
    """2049 tokens over a table of 2^21 pages pass the places that the attention kernel counts in 32 bits: the step is
    refused before the parent that it would consume is released."""
    s = pkg.DeviceSession(store, tiny(pkg, 1 << 25), 3, 2 << 30).kv4(track=True)
    (a,), _, _ = s.step_ragged([None], [0], [3], prompt(3))
    before = s.kv4_read(a, 0, weights=True)
    with pytest.raises(pkg.NativeError, match="split the call"):
        s.step_ragged([a], [3], [2049], prompt(2049, 2), flags=pkg.RAGGED_SAMPLED | pkg.RAGGED_CONSUME)
    assert all(np.array_equal(x, y) for x, y in zip(before, s.kv4_read(a, 0, weights=True)))
    (b,), _, _ = s.step_ragged([a], [3], [100], prompt(100, 3), flags=pkg.RAGGED_SAMPLED | pkg.RAGGED_CONSUME)
    assert s.kv4_read(b, 0)[0].shape[1] == 103
    assert s.drain() == 1
    s.close()


@pytest.mark.gpu
def test_a_session_that_cannot_track_keeps_its_pages(pkg, store):
    """Weights of 6000 slots of 2^22 tokens (201 GB) fit the byte budget and not the device: refused, and the session
    goes on with bf16 pages, or with 4-bit pages that do not track."""
    s = pkg.DeviceSession(store, tiny(pkg, 1 << 22), 6000, 1 << 38)
    with pytest.raises(pkg.NativeError, match="no device memory"):
        s.kv4(track=True)
    toks = prompt(20)
    (a,), first, _ = s.step_ragged([None], [0], [20], toks)
    with pytest.raises(pkg.NativeError, match="not 4-bit"):
        s.kv4_read(a, 0)
    s.release(a)
    s.kv4()
    (a,), _, _ = s.step_ragged([None], [0], [20], toks)
    k, v, _ = s.kv4_read(a, 0)
    assert k.shape == (KV_HEADS, 20, DIM) and np.isfinite(k).all() and np.isfinite(v).all() and k.any() and v.any()
    assert s.drain() == 1
    s.close()


@pytest.mark.gpu
@pytest.mark.parametrize("kv4", [False, True])
def test_draft_pool_holds_no_more_than_the_slots_can(pkg, make, store, kv4):
    """The draft head's bf16 pages: a context for each of 24 slots (6.3 MB), not one for every page of the target's
    pool (256 MB in bf16, 955 MB beside 4-bit pages)."""
    s = make(kv4)
    free = torch.cuda.mem_get_info()[0]
    s.mtp_attach(store)
    # beside it block tables, hidden rows and weights' scratch: a few MB, in allocations of 2 MB granularity
    assert free - torch.cuda.mem_get_info()[0] <= 32 << 20
    (a,), _, _ = s.step_ragged([None], [0], [40], prompt(40), flags=pkg.RAGGED_SAMPLED)
    s.release(a)


@pytest.mark.gpu
@pytest.mark.parametrize("track", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim,rope", [(4, 2, 128, 32), (6, 1, 64, 64)])
def test_other_heads_against_the_oracle(pkg, O, heads, kv_heads, dim, rope, track):
    """A prompt of 700 tokens in one step (several tokens per CTA of the append, split projection sums and gates), a
    block of 40 (128-row tiles of fp16 rows without tracking) and single tokens."""
    if not has_cuda():
        pytest.skip("no CUDA device")
    O.set_routing_slack(5e-2)

    def config(mod):
        return mod.config(hidden=256, layers=4, vocab=4096, q_heads=heads, kv_heads=kv_heads, head_dim=dim, key_heads=2,
                          value_heads=4, key_dim=64, value_dim=64, experts=16, top=2, intermediate=128, shared=128,
                          context=1024, rope_dims=rope, theta=THETA)

    store = pkg.WeightStore().synthetic(config(pkg), SEED)
    s = pkg.DeviceSession(store, config(pkg), slots=4, budget_bytes=1 << 28).kv4(track)
    model = O.Model(config(O), SEED)
    try:
        s.set_capture(True)
        toks = prompt(742, 21)
        cur, state, pos = None, None, 0
        for n in (700, 40, 1, 1):
            (cur,), _, logits = s.step_ragged([cur], [pos], [n], toks[pos:pos + n],
                                              flags=pkg.RAGGED_LOGITS | pkg.RAGGED_ALL_ROWS)
            route = s.debug_routing(n)
            held = np.stack(s.kv4_read(cur, 0)[:2])[None, :, :, pos:]
            lg, _, _, _ = model.forward(toks[pos:pos + n], pos, old_state=state, forced_routing=route, cached_kv=held)
            assert max(rel_l2(logits[j], lg[j]) for j in range(n)) <= 1e-2  # the tolerance of the bf16 sessions
            state, pos = s.snapshot(cur), pos + n
        if track:
            w = s.kv4_read(cur, 0, weights=True)[2]
            g = heads // kv_heads
            assert (abs(w.sum(1, dtype=np.float64) - g * pos) <= (WEIGHT_TOL * dim / 64 + g * pos * 2.0 ** -24) * g * pos).all()
        s.release(cur)
    finally:
        s.close()
        store.close()
