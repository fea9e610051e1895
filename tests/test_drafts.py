"""Sampled and speculated decoding without a GPU: the host functions, and every
argument that the entry points refuse before they touch the device (the context
handed in is a block of zeros that no refused call reads)."""
import ctypes as C

import numpy as np
import pytest

import drafts


@pytest.fixture
def fake():
    return C.cast(C.create_string_buffer(4096), C.c_void_p)


P = 1 << 20  # an aligned address that no refused call reads


def refused(lrs, rc, code, text):
    assert rc == code
    assert text in lrs.lib.lrs_last_error().decode()


@pytest.mark.parametrize("opt,text", [
    (dict(temperature=-0.1), "temperature"), (dict(temperature=float("nan")), "temperature"),
    (dict(temperature=float("inf")), "temperature"), (dict(top_p=1.5), "top_p"),
    (dict(top_p=float("nan")), "top_p"), (dict(top_p=-0.5), "top_p"), (dict(min_p=2.0), "min_p"),
    (dict(min_p=float("nan")), "min_p")])
def test_sampling_parameters_are_checked(lrs, fake, opt, text):
    refused(lrs, lrs.lib.lrs_sample_dev(fake, P, 100, 1, 100, C.byref(lrs.sampling(**opt)), P, P, None), -1, text)


@pytest.mark.parametrize("ld,rows,vocab,text", [
    (99, 1, 100, "ld"), (100, 0, 100, "rows"), (100, 65536, 100, "rows"), (100, 1, 0, "vocab"),
    (1 << 22, 1, (1 << 21) + 1, "vocab")])
def test_sample_shapes_are_checked(lrs, fake, ld, rows, vocab, text):
    s = C.byref(lrs.sampling())
    refused(lrs, lrs.lib.lrs_sample_dev(fake, P, ld, rows, vocab, s, P, P, None), -1, text)


def test_null_arguments(lrs, fake):
    s = C.byref(lrs.sampling())
    for a in ((None, P, 8, 1, 8, s, P, P, None), (fake, None, 8, 1, 8, s, P, P, None),
              (fake, P, 8, 1, 8, None, P, P, None), (fake, P, 8, 1, 8, s, None, P, None),
              (fake, P, 8, 1, 8, s, P, None, None)):
        refused(lrs, lrs.lib.lrs_sample_dev(*a), -1, "null")
    import llama_rs_amd.model  # binds the model's entry points
    L = lrs.lib
    refused(lrs, L.lrs_decode_sample(None, 0, 0, s, 0.5, None), -1, "null")
    refused(lrs, L.lrs_generate_sample(None, P, 1, 0, 1, s, P, P), -1, "null")
    refused(lrs, L.lrs_decode_tree(None, P, P, 1, 0, None), -1, "null")
    refused(lrs, L.lrs_tree_keep(None, P, 1), -1, "null")
    refused(lrs, L.lrs_verify_tree(None, P, P, 1, 0, s, P, P, None), -1, "null")


def kv(lrs, k=P, v=P, n_kv=2, rows=64, head_dim=128):
    return C.byref(lrs.LrsKv(k, v, n_kv, rows, head_dim))


@pytest.mark.parametrize("cache,n,n_head,code,text", [
    (dict(k=None), 1, 4, -1, "null"), (dict(v=None), 1, 4, -1, "null"), (dict(head_dim=96), 1, 4, -5, "head_dim"),
    (dict(n_kv=0), 1, 4, -1, "empty"), (dict(rows=0), 1, 4, -1, "empty"), (dict(), 0, 4, -1, "empty"),
    (dict(), 1, 5, -1, "multiple"), (dict(), 1, 0, -1, "multiple"), (dict(k=P + 8), 1, 4, -1, "aligned"),
    (dict(rows=1 << 31), 1, 4, -1, "rows"), (dict(), 1, 2048, -5, "heads")])
def test_caches_are_checked(lrs, fake, cache, n, n_head, code, text):
    L, r = lrs.lib, C.byref(lrs.LrsRope(64, 0, 0, 1.0))
    refused(lrs, L.lrs_attn_tree_dev(fake, kv(lrs, **cache), P, n, n_head, 3, None, 1.0, P), code, text)
    big = 1 << 20
    refused(lrs, L.lrs_rope_append_dev(fake, kv(lrs, **cache), r, P, P, big, P, big, P, big, P, P, n, n_head, 2 * P),
            code, text)


def test_attn_tree_arguments(lrs, fake):
    L = lrs.lib
    refused(lrs, L.lrs_attn_tree_dev(fake, kv(lrs), P, 4, 4, 61, None, 1.0, P), -4, "exceeds")
    refused(lrs, L.lrs_attn_tree_dev(fake, kv(lrs), P, 4, 4, 0xFFFFFFFE, None, 1.0, P), -4, "exceeds")
    refused(lrs, L.lrs_attn_tree_dev(fake, kv(lrs, rows=4096), P, 513, 4, 0, None, 1.0, P), -1, "512")
    refused(lrs, L.lrs_attn_tree_dev(fake, kv(lrs), P, 4, 4, 0, None, float("nan"), P), -1, "scale")
    refused(lrs, L.lrs_attn_tree_dev(fake, kv(lrs), P + 4, 4, 4, 0, None, 1.0, P), -1, "aligned")
    refused(lrs, L.lrs_attn_tree_dev(fake, kv(lrs), P, 4, 4, 0, None, 1.0, P + 4), -1, "aligned")
    refused(lrs, L.lrs_attn_tree_dev(fake, kv(lrs), P, 4, 4, 0, None, 1.0, P), -1, "the same")


def test_rope_append_arguments(lrs, fake):
    def call(rope_dim=64, layout=0, scale=1.0, freq=P, ldq=512, ldk=256, ldv=256, n=2, q=P, out=2 * P):
        r = C.byref(lrs.LrsRope(rope_dim, layout, 0, scale))
        return lrs.lib.lrs_rope_append_dev(fake, kv(lrs), r, freq, q, ldq, P, ldk, P, ldv, P, P, n, 4, out)

    refused(lrs, call(rope_dim=130), -1, "rope_dim")
    refused(lrs, call(rope_dim=63), -1, "rope_dim")
    refused(lrs, call(layout=2), -1, "layout")
    refused(lrs, call(scale=float("inf")), -1, "scale")
    refused(lrs, call(freq=None), -1, "freq")
    refused(lrs, call(ldq=511), -1, "stride")
    refused(lrs, call(ldk=255), -1, "stride")
    refused(lrs, call(ldv=255), -1, "stride")
    refused(lrs, call(n=65536), -1, "65535")
    refused(lrs, call(ldq=1024, out=P), -1, "dense")


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 100, 512])
def test_tree_mask(lrs, n):
    parents = drafts.random_tree(np.random.default_rng(n), n)
    if n > 40:
        parents[20] = -1  # a second root
    mask, depth = lrs.tree_mask(parents)
    seen = drafts.ancestors(parents)
    assert np.array_equal(mask, drafts.mask_words(seen))
    assert np.array_equal(depth, seen.sum(1) - 1)


@pytest.mark.parametrize("parents", [[], [0], [-1, 1], [-1, 0, 3, 0], [-1] * 513])
def test_bad_trees_are_refused(lrs, parents):
    with pytest.raises(lrs.ModelError) as e:
        lrs.tree_mask(parents)
    assert e.value.code == -1


@pytest.mark.parametrize("dim,base", [(128, 1e6), (64, 1e4), (2, 5e5), (250, 1e7)])
def test_rope_freqs(lrs, dim, base):
    i = np.arange(dim // 2)
    f, s = lrs.rope_freqs(dim, base)
    want = np.float64(np.float32(base)) ** (-2.0 * i / dim)
    half = 2.0 ** -24 * (1 + 1e-6)  # one rounding to f32
    assert s == 1.0 and np.all(np.abs(f - want) <= half * want)
    f, s = lrs.rope_freqs(dim, base, "linear", 4.0)
    assert s == 1.0 and np.all(np.abs(f - want / 4) <= half * want / 4)
    f, s = lrs.rope_freqs(dim, base, "yarn", 8.0, 4096)
    # pairs with more than 32 turns over 4096 positions stay, with less than
    # one turn all of factor 8; monotone between (the ramp's ends are whole pairs)
    turns = 4096 * want / (2 * np.pi)
    keep, slow = turns > 33 * base ** (2 / dim), turns < 0.99 * base ** (-2 / dim)
    assert np.all(np.abs(f - want)[keep] <= half * want[keep])
    assert np.all(np.abs(f - want / 8)[slow] <= half * want[slow] / 8)
    assert np.all(np.diff(f) < 0) and np.all(f <= want * (1 + half)) and np.all(f >= want / 8 * (1 - half))
    assert abs(s - (1 + 0.1 * np.log(8.0))) <= 2.0 ** -24 * s


@pytest.mark.parametrize("kw", [dict(rope_dim=0), dict(rope_dim=7), dict(rope_dim=258), dict(base=1.0),
                                dict(base=float("inf")), dict(scaling="linear", factor=0.5),
                                dict(scaling="yarn", factor=2.0), dict(scaling="other"),
                                dict(scaling="yarn", factor=2.0, orig_ctx=10, beta_fast=1.0)])
def test_rope_freqs_refusals(lrs, kw):
    a = dict(dict(rope_dim=64, base=1e4), **kw)
    with pytest.raises(lrs.ModelError) as e:
        lrs.rope_freqs(**a)
    assert e.value.code == -1


def test_wrappers_refuse_mismatched_sizes(lrs):
    class B:
        ptr, nbytes = P, 100

    with pytest.raises(lrs.ModelError):
        lrs.KvCache(B, B, 1, 64, 64)
    with pytest.raises(lrs.ModelError):
        lrs.sample(None, np.zeros((2, 5)), np.zeros(3))
    with pytest.raises(lrs.ModelError):
        lrs.sampling(top_k=-1)
