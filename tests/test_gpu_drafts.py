"""Sampled and speculated decoding on the GPU: the kernel-level operators
against their definitions in 64 bits (drafts.py), and the model's calls against
its own token-by-token decode."""
import numpy as np
import pytest

import drafts
import modelgen

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx(lrs):
    c = lrs.Context(0)
    yield c
    c.close()


def up(ctx, a):
    a = np.ascontiguousarray(a)
    b = ctx.alloc(max(a.nbytes, 16))
    b.upload(a)
    return b


def words(ctx, a):
    return up(ctx, np.asarray(a, np.int64).astype(np.uint32))


# ---------------------------------------------------------------------------
# sampling
# ---------------------------------------------------------------------------
def check_rows(tok, prob, x, u, opt):
    # a probability: one rounding to f32, weights to 2^-43 of the largest each
    for r in range(len(u)):
        t, p, kept = drafts.sample_row(x[r], u[r], **opt)
        assert int(tok[r]) == t, (r, int(tok[r]), t, kept.size, opt)
        assert abs(float(prob[r]) - p) <= 2.0 ** -23 * p + 2.0 ** -43 * (1 + kept.size * p), (r, prob[r], p)


def logits(rng, rows, vocab, quant=0):
    x = (2.2 * rng.standard_normal((rows, vocab))).astype(np.float32)
    top = rng.integers(0, vocab, (rows, min(40, vocab)))
    np.put_along_axis(x, top, rng.uniform(5, 14, top.shape).astype(np.float32), 1)
    return np.round(x * quant) / quant if quant else x


OPTS = [
    dict(temperature=0.0), dict(temperature=0.8, top_k=40, top_p=0.95, min_p=0.05), dict(temperature=1.0, top_k=1),
    dict(temperature=0.7, top_k=128), dict(temperature=0.7, top_k=128, top_p=0.5), dict(temperature=1.0, top_k=129),
    dict(temperature=1.0), dict(temperature=1.0, top_p=0.9), dict(temperature=1.3, top_k=500, top_p=0.98, min_p=0.01),
    dict(temperature=1.0, min_p=0.1), dict(temperature=3.0, top_p=0.7), dict(temperature=0.05, top_p=0.999),
    dict(temperature=1.0, top_p=0.0), dict(temperature=1.0, top_k=300, top_p=0.3), dict(temperature=1.0, min_p=1.0),
    dict(temperature=1e-30, top_k=50), dict(temperature=1e-30, top_p=0.9), dict(temperature=1e30, top_k=200),
    dict(temperature=1e30, top_p=0.5)]


@pytest.mark.parametrize("vocab", [1, 3, 127, 1000, 1024, 4099, 32000, 70001, 152064])
def test_sample_matches_definition(lrs, ctx, vocab):
    rng = np.random.default_rng(vocab)
    rows = 5 if vocab < 50000 else 3
    for quant in (0, 8):  # 8: many equal logits
        x = logits(rng, rows, vocab, quant)
        for opt in OPTS:
            print(f"vocab {vocab} quant {quant} {opt}", flush=True)
            u = rng.random(rows).astype(np.float32)
            tok, prob = lrs.sample(ctx, x, u, **opt)
            check_rows(tok, prob, x, u, opt)


@pytest.mark.parametrize("opt", OPTS, ids=lambda o: "-".join(f"{k[-1]}{v}" for k, v in o.items()))
def test_sample_odd_rows(lrs, ctx, opt):
    """masked words, NaN, infinities, ties, single words, nothing at all"""
    V = 5000
    rng = np.random.default_rng(3)
    x = logits(rng, 16, V)
    x[0] = -np.inf
    x[1] = np.nan
    x[2, :] = -np.inf
    x[2, 4321] = -1e30
    x[3, rng.random(V) < 0.95] = -np.inf
    x[4, rng.random(V) < 0.3] = np.nan
    x[5] = 0.25  # every word equal
    x[6, 77] = np.inf
    x[7, [5, 99, 4999]] = np.inf
    x[8] = np.where(rng.random(V) < 0.5, np.float32(-0.0), np.float32(0.0))
    x[9, :] = -3.0e38
    x[9, 1] = 3.0e38
    x[10] = np.arange(V) * 1e-3  # the largest last, in a few parts
    x[11] = -np.arange(V) * 1e-3
    x[12] = 1e-40 * np.arange(V)  # denormal steps
    x[13, :] = -np.inf
    x[13, :3] = [1.0, np.nan, 1.0]
    x[14] = np.where(np.arange(V) % 7 == 0, 8.0, -8.0)
    x[15, 0] = 60.0  # one word has all the mass
    u = rng.random(16).astype(np.float32)
    tok, prob = lrs.sample(ctx, x, u, **opt)
    check_rows(tok, prob, x, u, opt)


def test_sample_equal_words_past_the_list(lrs, ctx):
    """more words share a cut's bin than a row's list holds"""
    V = 40000
    x = np.zeros((4, V), np.float32)
    x[1, 17] = 50.0
    x[2, 1::2] = -1.0
    x[3] = np.arange(V) % 2 * 1e-6
    u = np.array([0.5, 0.1, 0.77, 0.999], np.float32)
    for opt in (dict(top_p=0.6), dict(top_k=9000), dict(top_k=20001, top_p=0.25), dict(top_k=30000, top_p=0.9, min_p=0.5)):
        print(opt, flush=True)
        tok, prob = lrs.sample(ctx, x, u, **opt)
        check_rows(tok, prob, x, u, opt)


@pytest.mark.parametrize("opt", [dict(top_k=129), dict(top_k=500), dict(top_k=500, top_p=0.5), dict(top_k=1024, min_p=0.5),
                                 dict(top_k=1024, top_p=0.9, min_p=0.01), dict(top_k=1025, top_p=0.9)],
                         ids=lambda o: "-".join(f"{k[-1]}{v}" for k, v in o.items()))
def test_sample_equal_words_around_a_rank(lrs, ctx, opt):
    """the last kept rank among more equal words than a row's list holds, and among fewer"""
    V = 40000
    rng = np.random.default_rng(44)
    x = np.zeros((6, V), np.float32)
    x[1, rng.permutation(V)[:300]] = 2.0
    x[2] = rng.integers(0, 4, V) * 0.25
    x[3] = -np.inf
    x[3, 7::100] = 1.0  # 400 words in all
    x[4, rng.permutation(V)[:1500]] = 4.0
    x[5] = np.where(np.arange(V) < 600, 1.0, -np.inf)
    u = np.array([0.0, 0.4, 0.71, 1.0 - 2.0 ** -24, np.nan, 0.9], np.float32)
    tok, prob = lrs.sample(ctx, x, u, **opt)
    check_rows(tok, prob, x, u, opt)


@pytest.mark.parametrize("opt", [dict(top_k=300), dict(top_k=700, top_p=0.95), dict(top_p=0.5), dict(min_p=0.02),
                                 dict(top_k=40, min_p=0.1)])
def test_sample_random_number_edges_of_each_form(lrs, ctx, opt):
    x = logits(np.random.default_rng(18), 1, 9001)[[0] * 8]
    u = np.array([0.0, -0.0, -3.0, np.nan, 1.0 - 2.0 ** -24, 1.0, np.inf, 2.0 ** -149], np.float32)
    tok, prob = lrs.sample(ctx, x, u, **opt)
    check_rows(tok, prob, x, u, opt)


@pytest.mark.parametrize("rows,vocab", [(700, 700), (300, 4500), (65, 33000)])
def test_sample_many_rows_of_each_form(lrs, ctx, rows, vocab):
    rng = np.random.default_rng(rows)
    x, u = logits(rng, rows, vocab), rng.random(rows).astype(np.float32)
    for opt in (dict(top_k=200, top_p=0.9), dict(top_k=1024), dict(top_p=0.8), dict(top_k=8, min_p=0.02)):
        tok, prob = lrs.sample(ctx, x, u, **opt)
        check_rows(tok, prob, x, u, opt)


@pytest.mark.parametrize("opt", [dict(top_k=20), dict(top_p=0.8), dict()])
def test_sample_random_number_edges(lrs, ctx, opt):
    x = logits(np.random.default_rng(8), 1, 3000)[[0] * 7]
    u = np.array([0.0, -0.0, -3.0, np.nan, 1.0 - 2.0 ** -24, 1.0, np.inf], np.float32)
    tok, prob = lrs.sample(ctx, x, u, **opt)
    check_rows(tok, prob, x, u, opt)


def test_sample_largest_vocabulary(lrs, ctx):
    V = 1 << 21
    x = logits(np.random.default_rng(9), 1, V)
    for opt in (dict(temperature=0.0), dict(top_k=30), dict(top_k=100), dict(top_p=0.9), dict()):
        tok, prob = lrs.sample(ctx, x, np.array([0.37], np.float32), **opt)
        check_rows(tok, prob, x, [0.37], opt)


@pytest.mark.parametrize("ld,shift", [(1003, 0), (1004, 1), (1008, 4)])
@pytest.mark.parametrize("opt", [dict(top_k=30, top_p=0.9), dict(top_p=0.9)])
def test_sample_strides_and_neighbours(lrs, ctx, ld, shift, opt):
    """rows of a wider matrix, unaligned; outputs behind the rows stay"""
    rng = np.random.default_rng(ld)
    buf = rng.standard_normal(7 * ld + shift).astype(np.float32) * 50
    x = buf[shift:].reshape(7, ld)[:, :1001]
    b = up(ctx, buf)

    class At:
        ptr = b.ptr + 4 * shift

    u = rng.random(7).astype(np.float32)
    ub, t, p = up(ctx, u), up(ctx, np.full(9, 5, np.uint32)), up(ctx, np.full(9, 5, np.float32))
    lrs.sample_dev(ctx, At, 7, 1001, ub, t, p, ld=ld, **opt)
    ctx.sync()
    tok, prob = t.download(np.uint32, 9), p.download(np.float32, 9)
    check_rows(tok, prob, x, u, opt)
    assert np.all(tok[7:] == 5) and np.all(prob[7:] == 5)
    lrs.sample_dev(ctx, At, 7, 1001, ub, t, None, ld=ld, **opt)  # no probabilities asked for
    ctx.sync()
    assert np.array_equal(t.download(np.uint32, 9), tok)


def test_sample_many_rows_and_repeats(lrs, ctx):
    """results do not depend on the rows beside, nor on the call"""
    rng = np.random.default_rng(21)
    x, u = logits(rng, 300, 2500), rng.random(300).astype(np.float32)
    for opt in (dict(top_k=50, top_p=0.9), dict(temperature=1.5, top_p=0.95)):
        tok, prob = lrs.sample(ctx, x, u, **opt)
        check_rows(tok, prob, x, u, opt)
        for i in (0, 299):
            t1, p1 = lrs.sample(ctx, x[i:i + 1], u[i:i + 1], **opt)
            assert t1[0] == tok[i] and p1[0] == prob[i]
        t2, p2 = lrs.sample(ctx, x, u, **opt)
        assert np.array_equal(tok, t2) and np.array_equal(prob, p2)


# ---------------------------------------------------------------------------
# rotation + append
# ---------------------------------------------------------------------------
ROPE = [  # n, n_head, n_kv, head_dim, rope_dim, halves
    (1, 40, 8, 128, 128, 0), (1, 1, 1, 64, 64, 1), (27, 24, 4, 256, 64, 1), (27, 24, 4, 256, 64, 0),
    (5, 7, 7, 64, 22, 0), (5, 7, 7, 64, 22, 1), (3, 6, 2, 128, 2, 1), (3, 6, 2, 128, 126, 0), (4, 8, 1, 256, 256, 1),
    (4, 8, 1, 256, 0, 0), (130, 10, 2, 128, 96, 1)]


def rope_bound(x, rope_dim, halves, scale):
    """an element's distance from the rotation's: cos and sin to 2^-22 (the angle,
    within pi, rounded to f32, then one ulp), two products and a sum of 2^-24
    each, over both elements' magnitudes"""
    return drafts_pair_sum(np.abs(x.astype(np.float64)), rope_dim, halves) * scale * (2.0 ** -22 + 4 * 2.0 ** -24)


def drafts_pair_sum(x, rope_dim, halves):
    i = np.arange(rope_dim // 2)
    a, b = (i, i + rope_dim // 2) if halves else (2 * i, 2 * i + 1)
    y = np.zeros_like(x)
    y[..., a] = y[..., b] = x[..., a] + x[..., b]
    return y


@pytest.mark.parametrize("n,n_head,n_kv,hd,rope_dim,halves", ROPE)
@pytest.mark.parametrize("pad,f32_angle", [(0, False), (4, False), (3, True)])
def test_rope_append(lrs, ctx, n, n_head, n_kv, hd, rope_dim, halves, pad, f32_angle):
    rng = np.random.default_rng([n, hd, rope_dim, pad])
    rows, scale = 300, 1.25 if pad else 1.0
    far = 4000 if f32_angle else (1 << 32) - 2
    q, k, v = (rng.standard_normal((n, h * hd + pad)).astype(np.float32) for h in (n_head, n_kv, n_kv))
    pos = rng.integers(0, far, n)
    pos[0], pos[-1] = 0 if n > 1 else 1711, pos[-1]
    slot = rng.permutation(rows)[:n]
    if n > 3:
        slot[2], slot[3] = 0xFFFFFFFF, rows  # padded tokens
    freq = np.float32(1e6) ** (-2.0 * np.arange(max(rope_dim // 2, 1)) / max(rope_dim, 1)).astype(np.float32)
    kc, vc = (rng.standard_normal((n_kv, rows, hd)).astype(np.float16) for _ in "kv")
    kb, vb, out = up(ctx, kc), up(ctx, vc), up(ctx, np.full((n + 1) * n_head * hd, 9, np.float32))
    lrs.rope_append_dev(ctx, lrs.KvCache(kb, vb, n_kv, rows, hd), up(ctx, freq), rope_dim, up(ctx, q), up(ctx, k),
                        up(ctx, v), words(ctx, pos), words(ctx, slot), n, n_head, out, layout=halves, scale=scale,
                        f32_angle=f32_angle, ldq=q.shape[1], ldk=k.shape[1], ldv=v.shape[1])
    ctx.sync()
    got = out.download(np.float32, (n + 1) * n_head * hd)
    assert np.all(got[n * n_head * hd:] == 9)
    qx = q[:, :n_head * hd].reshape(n, n_head, hd)
    want = drafts.rotate(qx, pos, freq, rope_dim, halves, scale, f32_angle)
    err = np.abs(got[:n * n_head * hd].reshape(n, n_head, hd) - want)
    assert np.all(err <= rope_bound(qx, rope_dim, halves, scale))
    kx = k[:, :n_kv * hd].reshape(n, n_kv, hd)
    kw = drafts.rotate(kx, pos, freq, rope_dim, halves, scale, f32_angle)
    kt = rope_bound(kx, rope_dim, halves, scale)
    kt = kt + 2.0 ** -11 * (np.abs(kw) + kt) + 2.0 ** -25  # the rounding to f16
    kg, vg = (b.download(np.float16, kc.size).reshape(kc.shape) for b in (kb, vb))
    vw = vc.copy()
    left = np.ones(rows, bool)
    for t in range(n):
        if slot[t] < rows:
            left[slot[t]] = False
            assert np.all(np.abs(kg[:, slot[t]].astype(np.float64) - kw[t]) <= kt[t])
            vw[:, slot[t]] = v[t, :n_kv * hd].reshape(n_kv, hd).astype(np.float16)
    assert np.array_equal(kg[:, left], kc[:, left])
    assert np.array_equal(vg, vw)


def test_rope_append_in_place(lrs, ctx):
    rng = np.random.default_rng(2)
    for rope_dim, halves in ((64, 1), (64, 0), (30, 1), (30, 0)):
        q, k = rng.standard_normal((6, 4 * 64)).astype(np.float32), rng.standard_normal((6, 64)).astype(np.float32)
        freq, pos = np.float32(0.5) ** np.arange(32, dtype=np.float32), np.arange(6) * 1000
        kb = up(ctx, np.zeros((1, 8, 64), np.float16))
        kv = lrs.KvCache(kb, up(ctx, np.zeros((1, 8, 64), np.float16)), 1, 8, 64)
        qb = up(ctx, q)
        lrs.rope_append_dev(ctx, kv, up(ctx, freq), rope_dim, qb, up(ctx, k), up(ctx, k), words(ctx, pos),
                            words(ctx, np.arange(6)), 6, 4, qb, layout=halves)
        ctx.sync()
        x = q.reshape(6, 4, 64)
        err = np.abs(qb.download(np.float32, q.size).reshape(x.shape) - drafts.rotate(x, pos, freq, rope_dim, halves))
        assert np.all(err <= rope_bound(x, rope_dim, halves, 1.0))


# ---------------------------------------------------------------------------
# attention of a tree
# ---------------------------------------------------------------------------
def attn(lrs, ctx, q, kc, vc, length, mask, scale=None):
    n, H, D = q.shape
    kv = lrs.KvCache(up(ctx, kc), up(ctx, vc), kc.shape[0], kc.shape[1], D)
    out = up(ctx, np.full((n + 1) * H * D, 7, np.float32))
    lrs.attn_tree_dev(ctx, kv, up(ctx, q), n, H, length, None if mask is None else up(ctx, mask), out, scale=scale)
    ctx.sync()
    got = out.download(np.float32, (n + 1) * H * D)
    assert np.all(got[n * H * D:] == 7)
    return got[:n * H * D].reshape(q.shape)


def attn_case(rng, n, H, G, D, rows):
    q = (1.5 * rng.standard_normal((n, H, D))).astype(np.float32)
    return (q, *(rng.standard_normal((G, rows, D)).astype(np.float16) for _ in "kv"))


ATTN = [  # n, n_head, n_kv, head_dim, len
    (1, 1, 1, 64, 0), (1, 8, 1, 128, 0), (1, 40, 8, 128, 1), (1, 6, 2, 256, 31), (8, 10, 2, 128, 333),
    (26, 10, 2, 128, 1000), (33, 5, 5, 64, 32), (41, 12, 2, 256, 95), (64, 10, 2, 128, 2047), (7, 24, 3, 64, 4097),
    (3, 33, 1, 128, 64), (100, 4, 4, 64, 17), (512, 2, 1, 64, 5), (5, 8, 8, 256, 5003), (2, 7, 1, 64, 20011)]


@pytest.mark.parametrize("n,H,G,D,length", ATTN)
def test_attn_tree(lrs, ctx, n, H, G, D, length):
    rng = np.random.default_rng([n, H, length])
    rows = length + n + int(rng.integers(0, 40))
    q, kc, vc = attn_case(rng, n, H, G, D, rows)
    kc[:, length + n:] = np.nan  # rows behind the tree are never read into a result
    vc[:, length + n:] = np.nan
    tree = drafts.ancestors(drafts.random_tree(rng, n))
    seen = np.concatenate([np.ones((n, length), bool), tree], 1)
    words_ = drafts.mask_words(tree)
    if n % 32:
        words_[:, -1] |= np.uint32(0xFFFFFFFF << (n % 32) & 0xFFFFFFFF)  # bits past the nodes mean nothing
    want, tol = drafts.attend(q, kc[:, :length + n], vc[:, :length + n], seen, D ** -0.5)
    got = attn(lrs, ctx, q, kc, vc, length, words_)
    assert np.all(np.abs(got - want) <= tol)
    chain = np.tril(np.ones((n, n), bool))
    seen = np.concatenate([np.ones((n, length), bool), chain], 1)
    want, tol = drafts.attend(q, kc[:, :length + n], vc[:, :length + n], seen, 0.3 * D ** -0.5)
    got = attn(lrs, ctx, q, kc, vc, length, None, scale=0.3 * D ** -0.5)
    assert np.all(np.abs(got - want) <= tol)


@pytest.mark.parametrize("n,G,length", [(9, 2, 0), (40, 1, 0), (9, 2, 50)])
def test_attn_tree_any_mask(lrs, ctx, n, G, length):
    """masks that are no tree, and rows that see nothing"""
    rng = np.random.default_rng(n)
    q, kc, vc = attn_case(rng, n, 4, G, 64, length + n)
    tree = rng.random((n, n)) < 0.3
    tree[3] = False
    seen = np.concatenate([np.ones((n, length), bool), tree], 1)
    want, tol = drafts.attend(q, kc, vc, seen, 0.125)
    got = attn(lrs, ctx, q, kc, vc, length, drafts.mask_words(tree))
    assert np.all(np.abs(got - want) <= tol)
    if length == 0:
        assert np.all(got[3] == 0)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("length", [0, 3, 70])
def test_attn_tree_unseen_values_do_not_leak(lrs, ctx, D, length):
    """NaN and infinities in K and V reach the rows that see them alone"""
    n, rng = 40, np.random.default_rng(D + length)
    q, kc, vc = attn_case(rng, n, 6, 2, D, length + n)
    tree = drafts.ancestors(drafts.random_tree(rng, n, 1.0))
    bad_v = {2: np.nan, 5: np.inf, 6: -np.inf, 33: np.nan}
    bad_k = {11: np.nan, 37: np.inf}
    clean_k, clean_v = kc.copy(), vc.copy()
    for j, x in bad_v.items():
        vc[:, length + j, ::3] = x
    for j, x in bad_k.items():
        kc[:, length + j, 1] = x
    got = attn(lrs, ctx, q, kc, vc, length, drafts.mask_words(tree))
    seen = np.concatenate([np.ones((n, length), bool), tree], 1)
    want, tol = drafts.attend(q, clean_k, clean_v, seen, D ** -0.5)
    sees = lambda j: tree[:, j]  # noqa: E731
    dirty_k = np.any([sees(j) for j in bad_k], 0)
    dirty_v = np.any([sees(j) for j in bad_v], 0) & ~dirty_k
    clean = ~dirty_k & ~dirty_v
    assert clean.sum() >= 3 and dirty_v.sum() >= 3
    assert np.all(np.abs(got - want)[clean] <= tol[clean])
    # the elements of V that are finite are right in the rows that see the others
    cols = np.arange(D) % 3 != 0
    assert np.all((np.abs(got - want) <= tol)[dirty_v][..., cols])
    for i in np.flatnonzero(dirty_v):
        bad = [x for j, x in bad_v.items() if tree[i, j]]
        x = got[i][:, ~cols]
        if any(np.isnan(b) for b in bad) or len(set(bad)) > 1:
            assert np.all(np.isnan(x))
        else:
            assert np.all(x == bad[0])


def test_attn_tree_large_scores(lrs, ctx):
    """one position far above the others, and all of them far below 0"""
    rng = np.random.default_rng(5)
    q, kc, vc = attn_case(rng, 3, 2, 1, 128, 700)
    q *= 40
    tree = np.eye(3, dtype=bool)
    seen = np.concatenate([np.ones((3, 697), bool), tree], 1)
    want, tol = drafts.attend(q, kc, vc, seen, 1.0)
    assert np.all(np.abs(attn(lrs, ctx, q, kc, vc, 697, drafts.mask_words(tree), 1.0) - want) <= tol)
    kc[..., 0], q[..., 0] = 1000, -1000
    want, tol = drafts.attend(q, kc, vc, seen, 1.0)
    assert np.all(np.abs(attn(lrs, ctx, q, kc, vc, 697, drafts.mask_words(tree), 1.0) - want) <= tol)


# ---------------------------------------------------------------------------
# together, captured
# ---------------------------------------------------------------------------
def test_operators_captured_and_replayed(lrs, ctx):
    """append, attention and two samplings recorded into graphs whose work they
    share; each replay, with other inputs, equals the eager calls"""
    rng = np.random.default_rng(77)
    n, H, G, D, L, V = 9, 10, 2, 128, 400, 6000
    kv = lrs.KvCache(up(ctx, rng.standard_normal((G, 512, D)).astype(np.float16)),
                     up(ctx, rng.standard_normal((G, 512, D)).astype(np.float16)), G, 512, D)
    tree = drafts.random_tree(rng, n)
    mask, depth = lrs.tree_mask(tree)
    freq, _ = lrs.rope_freqs(D, 1e6)
    fb, mb, pos, slot = up(ctx, freq), up(ctx, mask), words(ctx, L + depth), words(ctx, L + np.arange(n))
    qb, kb, vb, qo, out = (ctx.alloc(4 * n * w * D) for w in (H, G, G, H, H))
    xb, ub, t1, t2, pb = ctx.alloc(4 * n * V), ctx.alloc(4 * n), ctx.alloc(4 * n), ctx.alloc(4 * n), ctx.alloc(4 * n)

    def attention():
        lrs.rope_append_dev(ctx, kv, fb, D, qb, kb, vb, pos, slot, n, H, qo)
        lrs.attn_tree_dev(ctx, kv, qo, n, H, L, mb, out)

    def picks():
        lrs.sample_dev(ctx, xb, n, V, ub, t1, pb, temperature=0.9, top_k=40, top_p=0.9)
        lrs.sample_dev(ctx, xb, n, V, ub, t2, temperature=1.1, top_p=0.9)

    def read():
        ctx.sync()
        return [b.download(np.uint32, b.nbytes // 4) for b in (qo, out, t1, t2, pb)]

    def fill(seed):
        r = np.random.default_rng(seed)
        for b, w in ((qb, H), (kb, G), (vb, G)):
            b.upload(r.standard_normal(n * w * D).astype(np.float32))
        xb.upload(logits(r, n, V))
        ub.upload(r.random(n).astype(np.float32))

    fill(0)
    attention(), picks()
    ctx.sync()
    g1, g2 = ctx.capture(attention), ctx.capture(picks)
    try:
        for seed in (1, 2, 3, 4):
            fill(seed)
            g1.launch(), g2.launch()
            got = read()
            for b in (qo, out, t1, t2, pb):
                b.upload(np.zeros(b.nbytes, np.uint8))
            attention(), picks()
            for a, b in zip(got, read()):
                assert np.array_equal(a, b), seed
    finally:
        g1.close(), g2.close()


# ---------------------------------------------------------------------------
# the model's calls
# ---------------------------------------------------------------------------
def rel_l2(a, b):
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    return float(np.linalg.norm(a - b) / np.linalg.norm(b))


@pytest.fixture(scope="module")
def dense(lrs, orc, ctx):
    cfg = modelgen.GQA5
    return modelgen.gpu_model(lrs, ctx, cfg, modelgen.host_model(orc, cfg, seed=11, mode=1)), cfg


def path_to(parents, i):
    p = []
    while i >= 0:
        p.append(i)
        i = parents[i]
    return p[::-1]


@pytest.mark.parametrize("n,pos0", [(1, 0), (1, 30), (7, 0), (13, 20), (40, 64), (33, 127)])
def test_decode_tree_matches_decode(dense, n, pos0):
    """every node's logits against the decode of its path, at the prompt path's
    bar; keeping a path leaves the cache that the decode leaves"""
    m, cfg = dense
    rng = np.random.default_rng([n, pos0])
    toks, ctx_toks = rng.integers(0, cfg["vocab"], n), rng.integers(0, cfg["vocab"], pos0)
    tree = drafts.random_tree(rng, n)
    m.reset()

    def history():
        for i, t in enumerate(ctx_toks):
            m.decode(t, i)

    history()
    got = m.decode_tree(toks, tree, pos0)
    assert len(m) == pos0
    deep = max(range(n), key=lambda i: len(path_to(tree, i)))
    keep = path_to(tree, deep)
    m.tree_keep(keep)
    assert len(m) == pos0 + len(keep)
    after = m.decode(3, len(m)) if len(m) < cfg["ctx"] else None
    for i in {0, n // 2, n - 1, deep}:
        path = path_to(tree, i)
        for d, j in enumerate(path):
            want = m.decode(toks[j], pos0 + d)
        assert rel_l2(got[i], want) < 1e-3, i
    if after is not None:
        for d, j in enumerate(keep):
            m.decode(toks[j], pos0 + d)
        assert rel_l2(after, m.decode(3, pos0 + len(keep))) < 1e-3


def test_tree_refusals(lrs, dense):
    m, cfg = dense
    m.reset()
    m.decode(1, 0)

    def code(f, *a, **k):
        with pytest.raises(lrs.ModelError) as e:
            f(*a, **k)
        return e.value.code

    assert code(m.tree_keep, [0]) == -1  # no tree
    assert code(m.decode_tree, [1, 2], [-1, 1], 1) == -1
    assert code(m.decode_tree, [1, cfg["vocab"]], [-1, 0], 1) == -1
    assert code(m.decode_tree, [1, 2], [-1, 0], cfg["ctx"] - 1) == -4
    assert code(m.decode_tree, [], [], 1) == -1
    assert code(m.verify_tree, [1, 2], [-1, -1], 1) == -1
    assert code(m.verify_tree, [1, 2], [-1, 0], 1, temperature=0.5) == -1
    assert code(m.verify_tree, [1, 2], [-1, 0], 1, u=[0.5, 0.5], top_p=7.0) == -1
    assert code(m.decode_sample, 1, 1, 0.5, temperature=-1.0) == -1
    assert code(m.decode_sample, cfg["vocab"], 1, 0.5) == -1
    assert code(m.generate_sample, [1], [0.5] * cfg["ctx"], 1) == -4
    assert len(m) == 1
    m.decode_tree([1, 2, 3], [-1, 0, 0], 1, logits=False)
    for bad in ([1], [0, 0], [0, 1, 2], [2, 0], [0, 3], []):
        assert code(m.tree_keep, bad) == -1
    m.decode(1, 1)
    assert code(m.tree_keep, [0]) == -1  # the decode has dropped the tree


@pytest.mark.parametrize("opt", [dict(temperature=0.0), dict(temperature=0.7, top_k=20, top_p=0.9),
                                 dict(temperature=1.2, top_p=0.8), dict(temperature=1.0)])
def test_decode_and_generate_sample(dense, opt):
    """tokens are the definition's on the logits that decode returns, one by one
    and in a chain"""
    m, cfg = dense
    rng = np.random.default_rng(12)
    prompt, u = rng.integers(0, cfg["vocab"], 9), rng.random(24).astype(np.float32)
    m.reset()
    for i, t in enumerate(prompt[:-1]):
        m.decode(t, i)
    tok, toks = int(prompt[-1]), []
    for i in range(24):
        pos = len(prompt) - 1 + i
        want = drafts.sample_row(m.decode(tok, pos), u[i], **opt)[0]
        assert m.decode_sample(tok, pos, u[i], **opt) == want, i
        tok = want
        toks.append(tok)
    assert m.generate_sample(prompt[-1:], u, pos0=len(prompt) - 1, **opt).tolist() == toks
    assert len(m) == len(prompt) + 23
    if opt["temperature"] == 0:
        assert m.generate_greedy(prompt[-1:], 24, len(prompt) - 1).tolist() == toks


@pytest.mark.parametrize("opt", [dict(), dict(temperature=0.6, top_k=30, top_p=0.9), dict(temperature=1.0, top_p=0.7)])
def test_verify_tree_is_decode_by_steps(dense, opt):
    """drafts that are partly right: the tokens are those that token-by-token
    decoding gives with the same random numbers, and the sequence goes on from
    the cache that the walk leaves"""
    m, cfg = dense
    rng = np.random.default_rng(31)
    prompt = rng.integers(0, cfg["vocab"], 17)
    u = rng.random(64).astype(np.float32)
    m.reset()
    m.decode_batch(prompt[:-1], 0)
    pos = len(prompt) - 1
    plain = opt.get("temperature", 0.0) == 0.0
    want = (m.generate_greedy(prompt[-1:], 40, pos) if plain else
            m.generate_sample(prompt[-1:], u[:40], pos, **opt)).tolist()
    m.reset()
    m.decode_batch(prompt[:-1], 0)
    last, got, sizes = int(prompt[-1]), [], []
    while len(got) < 34:
        # the right continuation for a few tokens, with wrong siblings around it
        right = want[len(got):len(got) + int(rng.integers(0, 6))]
        toks, parents, depth, cur = [last], [-1], [0], 0
        for t in right:
            wrong = int((t + 1 + rng.integers(0, 50)) % cfg["vocab"])
            for x in ((wrong, t) if rng.random() < 0.5 else (t, wrong)):
                toks.append(x)
                parents.append(cur)
                depth.append(depth[cur] + 1)
            cur = len(toks) - (1 if toks[-1] == t else 2)
        un = None if plain else u[len(got) + np.array(depth)]
        out = m.verify_tree(toks, parents, pos, un, **opt).tolist()
        assert out[:-1] == right and len(out) == len(right) + 1
        got += out
        sizes.append(len(out))
        pos += len(out)
        assert len(m) == pos
        last = got[-1]
    assert got == want[:len(got)]
    assert max(sizes) > 3


def test_samplers_of_a_hybrid_model(lrs, orc, ctx):
    cfg = modelgen.HY_TINY
    m = modelgen.gpu_hybrid_model(lrs, ctx, cfg, modelgen.hybrid_host_model(orc, cfg, seed=3))
    opt = dict(temperature=0.8, top_k=25, top_p=0.95)
    u = np.random.default_rng(4).random(12).astype(np.float32)
    want, tok = [], 5
    for i in range(12):
        tok = drafts.sample_row(m.decode(tok, i), u[i], **opt)[0]
        want.append(tok)
    m.reset()
    assert m.generate_sample([5], u, **opt).tolist() == want
    m.reset()
    assert m.decode_sample(5, 0, u[0], **opt) == want[0]
    with pytest.raises(lrs.ModelError) as e:
        m.decode_tree([1, 2], [-1, 0], 1)
    assert e.value.code == -5
    m.close()


def test_logits_without_a_word(lrs, orc, ctx):
    """a head whose logits are all NaN: an error, and the state says what is cached"""
    def broken(w):
        t, a = w["output"]
        assert t == lrs.Q6_K
        a = np.array(a, copy=True)
        blocks = a.reshape(-1).view(np.uint8).reshape(-1, 210)
        blocks[:, 208:] = np.frombuffer(np.float16(np.nan).tobytes(), np.uint8)
        return dict(w, output=(t, a))

    def fails(f, *a, **k):
        with pytest.raises(lrs.ModelError) as e:
            f(*a, **k)
        assert e.value.code == -2 and "sampled" in str(e.value)

    m = modelgen.gpu_model(lrs, ctx, modelgen.GQA5, broken(modelgen.host_model(orc, modelgen.GQA5, seed=11, mode=1)))
    assert np.isnan(m.decode(3, 0)).all()
    for opt in (dict(temperature=0.0), dict(top_k=10), dict(top_p=0.9)):
        fails(m.decode_sample, 4, 1, 0.5, **opt)
        assert len(m) == 2
        fails(m.generate_sample, [4, 5, 6], [0.5] * 4, 1, **opt)
        assert len(m) == 4
        fails(m.verify_tree, [4, 5, 6], [-1, 0, 0], 1, u=[0.5] * 3, **opt)
        assert len(m) == 1
    m.close()
    cfg = modelgen.HY_TINY
    m = modelgen.gpu_hybrid_model(lrs, ctx, cfg, broken(modelgen.hybrid_host_model(orc, cfg, seed=3)))
    fails(m.decode_sample, 4, 0, 0.5)
    assert len(m) == 1
    fails(m.generate_sample, [4, 5], [0.5] * 4, 1)
    assert len(m) == 0
    m.close()
