"""The operators of sampled and speculated decoding: what is measured of them.

  rope_append  q and k of n tokens rotated at given positions, k and v rounded
               to f16 into given slots of the cache
  attn_tree    attention of n drafted tokens over the cache and over those of
               the n that a bit mask lets each of them see
  sample       one token of each row of logits from a given random number:
               temperature, top-k, top-p, min-p

Head counts, head widths and vocabularies are those of the dense and the
hybrid model's configurations (40 / 8 heads of 128, 24 / 4 heads of 256;
32000, 152064 and 248320 words) and a generic one of 64-wide heads; contexts
run from none to 131072 positions.  The cache is [n_kv][rows][head_dim] in
f16, activations and logits are f32.  `own` says whether run() calls this
package's operators or computes the same in elementary torch operations.
"""
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False
DEV = "cuda"
PAIRS, HALVES = 0, 1


def _product():
    """The package (its folder's name is no Python identifier)."""
    if "llama_rs_amd" not in sys.modules:
        pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llama.rs_amd")
        spec = importlib.util.spec_from_file_location(
            "llama_rs_amd", os.path.join(pkg, "__init__.py"), submodule_search_locations=[pkg])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["llama_rs_amd"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["llama_rs_amd"]


_ctx = None


def _context():
    global _ctx
    if _ctx is None:
        _ctx = _product().Context(0)
    return _ctx


class _Buf:
    """A torch tensor as the device buffer that the *_dev calls take."""

    def __init__(self, t):
        self.ptr, self.nbytes = t.data_ptr(), t.numel() * t.element_size()


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # the token of one decode step of a small vocabulary, the usual
        # truncations of a chat: launch latency is all there is
        dict(name="sample_chat_32k", kind="sample", rows=1, vocab=32000, temp=0.8, top_k=40, top_p=0.95,
             min_p=0.05, masked=0.0),
        # ... of the dense model's vocabulary with a nucleus alone: how many
        # words are kept is up to the logits
        dict(name="sample_nucleus_152k", kind="sample", rows=1, vocab=152064, temp=1.0, top_k=0, top_p=0.9,
             min_p=0.0, masked=0.0),
        # the nodes of a verified tree, each with its own sample
        dict(name="sample_tree_152k", kind="sample", rows=25, vocab=152064, temp=0.7, top_k=50, top_p=0.9,
             min_p=0.0, masked=0.0),
        # many rows of the widest vocabulary at a high temperature, most of a
        # grammar's words masked with -inf, a nucleus inside a wide top-k
        dict(name="sample_wide_248k", kind="sample", rows=64, vocab=248320, temp=1.3, top_k=1000, top_p=0.98,
             min_p=0.01, masked=0.5),
        # one token of the dense model
        dict(name="rope_append_1", kind="rope", n=1, n_head=40, n_kv=8, head_dim=128, rope_dim=128, layout=PAIRS,
             base=1e6, stretch=1.0, rows=4096, first=1711),
        # a drafted tree of the hybrid's attention shape, a quarter of the head rotated
        dict(name="rope_append_tree", kind="rope", n=27, n_head=24, n_kv=4, head_dim=256, rope_dim=64,
             layout=HALVES, base=1e7, stretch=1.0, rows=4096, first=3333),
        # a prompt block far into a stretched context
        dict(name="rope_append_512", kind="rope", n=512, n_head=40, n_kv=8, head_dim=128, rope_dim=128,
             layout=HALVES, base=1e6, stretch=4.0, rows=131072, first=129999),
        # a few drafted tokens in a short conversation of the dense model
        dict(name="attn_tree_8_short", kind="attn", n=8, n_head=40, n_kv=8, head_dim=128, len=333),
        # a tree near the end of the dense model's 4096 positions
        dict(name="attn_tree_26", kind="attn", n=26, n_head=40, n_kv=8, head_dim=128, len=3900),
        # the hybrid's attention shape
        dict(name="attn_tree_41_hd256", kind="attn", n=41, n_head=24, n_kv=4, head_dim=256, len=2047),
        # a draft of five behind a long document, narrow heads
        dict(name="attn_tree_5_32k", kind="attn", n=5, n_head=32, n_kv=8, head_dim=64, len=32768),
        # a wide tree behind a very long document (the largest case)
        dict(name="attn_tree_64_130k", kind="attn", n=64, n_head=40, n_kv=8, head_dim=128, len=130000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["sample", "rope", "attn"])
    if kind == "sample":
        return dict(kind=kind, rows=_log(rng, 1, 64), vocab=_log(rng, 500, 248320), temp=round(rng.uniform(0.3, 1.5), 3),
                    top_k=rng.choice([0, _log(rng, 1, 128), _log(rng, 1, 5000)]),
                    top_p=rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]),
                    min_p=rng.choice([0.0, round(rng.uniform(0.005, 0.3), 3)]), masked=rng.choice([0.0, 0.3, 0.9]))
    n_kv, rep, hd = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 5, 6, 7, 8]), rng.choice([64, 128, 256])
    if kind == "rope":
        rows = _log(rng, 2000, 131072)
        n = _log(rng, 1, 512)
        return dict(kind=kind, n=n, n_head=n_kv * rep, n_kv=n_kv, head_dim=hd, rope_dim=2 * rng.randint(1, hd // 2),
                    layout=rng.choice([PAIRS, HALVES]), base=rng.choice([1e4, 1e6, 1e7]),
                    stretch=rng.choice([1.0, 4.0]), rows=rows, first=rng.randint(0, rows - n))
    n_kv, n = min(n_kv, 1024 // hd), _log(rng, 1, 64)
    return dict(kind=kind, n=n, n_head=n_kv * min(rep, 5), n_kv=n_kv, head_dim=hd,
                len=rng.choice([0, _log(rng, 1, 4096), _log(rng, 100, 130000), _log(rng, 100, 130000)]))


# ---------------------------------------------------------------------------
# what a program has before the call
# ---------------------------------------------------------------------------
def _gen(seed, *path):
    """A generator of its own for every tensor of a seed."""
    h = int(seed) & 0xFFFFFFFFFFFF
    for p in path:
        h = (h * 1000003 + p + 1) % (1 << 61)
    g = torch.Generator(device=DEV)
    g.manual_seed(h)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _tree(seed, n):
    """parents [n] of a tree of drafts: node 0 is the root, the next level's
    nodes hang mostly below the likelier (earlier) nodes."""
    r = np.random.default_rng([seed, n])
    return [-1] + [int(i * r.random() ** 1.5) for i in range(1, n)]


def _ancestors(parents):
    n = len(parents)
    a = np.zeros((n, n), bool)
    for i, p in enumerate(parents):
        if p >= 0:
            a[i] = a[p]
        a[i, i] = True
    return a


def _words(a):
    """bit j of a row's words: whether the node sees node j"""
    n = a.shape[0]
    w = (n + 31) // 32
    b = np.zeros((n, 32 * w), np.uint64)
    b[:, :n] = a
    return (b.reshape(n, w, 32) << np.arange(32, dtype=np.uint64)).sum(2).astype(np.uint32).view(np.int32)


def _freq(case):
    """base^(-2i / rope_dim), positions stretched: the program's table"""
    i = np.arange(case["rope_dim"] // 2, dtype=np.float64)
    f = case["base"] ** (-2.0 * i / case["rope_dim"]) / case["stretch"]
    return torch.from_numpy(f.astype(np.float32)).to(DEV)


def prepare(case, seed):
    k = case["kind"]
    if k == "sample":
        rows, V = case["rows"], case["vocab"]
        # logits of a language model: a broad bulk, a few dozen words that
        # stand out, a grammar's masked words
        x = 2.2 * _randn(_gen(seed, 0), rows, V)
        top = torch.randint(0, V, (rows, 40), generator=_gen(seed, 1), device=DEV)
        lift = 6.0 + 9.0 * torch.rand(rows, 40, generator=_gen(seed, 2), device=DEV) ** 2
        x.scatter_(1, top, lift)
        if case["masked"]:
            x.masked_fill_(torch.rand(rows, V, generator=_gen(seed, 3), device=DEV) < case["masked"], -math.inf)
            x[:, V // 2] = 1.0  # a word that the grammar always allows
        s = dict(case=case, logits=x, u=torch.rand(rows, generator=_gen(seed, 4), device=DEV),
                 tokens=torch.empty(rows, dtype=torch.int32, device=DEV), probs=torch.empty(rows, device=DEV))
    else:
        n, H, G, D = case["n"], case["n_head"], case["n_kv"], case["head_dim"]
        rows = case["rows"] if k == "rope" else case["len"] + n
        s = dict(case=case, q=_randn(_gen(seed, 0), n, H * D), out=torch.empty(n, H * D, device=DEV),
                 kc=_randn(_gen(seed, 1), G, rows, D).half(), vc=_randn(_gen(seed, 2), G, rows, D).half())
        parents = _tree(seed, n)
        seen = _ancestors(parents)
        if k == "rope":
            s["k"], s["v"] = _randn(_gen(seed, 3), n, G * D), _randn(_gen(seed, 4), n, G * D)
            # a block of a prompt: consecutive positions; a tree: position by depth, slots in a row
            depth = np.arange(n) if n > 64 else seen.sum(1) - 1
            s["pos"] = torch.from_numpy((case["first"] + depth).astype(np.int32)).to(DEV)
            s["slot"] = torch.arange(case["first"], case["first"] + n, dtype=torch.int32, device=DEV)
            s["freq"] = _freq(case)
        else:
            s["q"] *= 1.5
            s["mask"] = torch.from_numpy(_words(seen)).to(DEV)
    s["bufs"] = {name: _Buf(t) for name, t in s.items() if torch.is_tensor(t)}
    torch.cuda.synchronize()
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    return {"sample": _sample, "rope": _rope_append, "attn": _attn_tree}[s["case"]["kind"]](s)


def _sample(s):
    c = s["case"]
    if own:
        b = s["bufs"]
        _product().sample_dev(_context(), b["logits"], c["rows"], c["vocab"], b["u"], b["tokens"], b["probs"],
                              temperature=c["temp"], top_k=c["top_k"], top_p=c["top_p"], min_p=c["min_p"])
        return s["tokens"], s["probs"]
    V = c["vocab"]
    k = min(c["top_k"], V) if c["top_k"] else V
    temp, top_p, min_p = (float(np.float32(c[x])) for x in ("temp", "top_p", "min_p"))
    # sums over a vocabulary next to a cut: in 64 bits
    x, idx = torch.sort(s["logits"], dim=1, descending=True, stable=True)
    w = torch.exp((x[:, :k].double() - x[:, :1].double()) / temp)
    sums = torch.cumsum(w, 1)
    kept = w >= min_p
    if top_p < 1.0:
        before = torch.cat([torch.zeros_like(sums[:, :1]), sums[:, :-1]], 1)
        kept &= before < top_p * sums[:, -1:]
    kept[:, 0] = True
    full = torch.zeros_like(s["logits"], dtype=torch.float64).scatter_(1, idx[:, :k], torch.where(kept, w, 0.0))
    sums = torch.cumsum(full, 1)
    tok = torch.searchsorted(sums, s["u"].double()[:, None] * sums[:, -1:], right=True)
    prob = full.gather(1, tok) / sums[:, -1:]
    return tok[:, 0].int(), prob[:, 0].float()


def _rope_append(s):
    c = s["case"]
    n, H, G, D = c["n"], c["n_head"], c["n_kv"], c["head_dim"]
    if own:
        lrs, b = _product(), s["bufs"]
        lrs.rope_append_dev(_context(), lrs.KvCache(b["kc"], b["vc"], G, c["rows"], D), b["freq"], c["rope_dim"],
                            b["q"], b["k"], b["v"], b["pos"], b["slot"], n, H, b["out"], layout=c["layout"])
        return s["out"], s["kc"], s["vc"]
    # angles of far positions: in 64 bits
    th = (s["pos"].double()[:, None] * s["freq"].double()[None, :])[:, None, :]
    cos, sin = torch.cos(th).float(), torch.sin(th).float()
    s["out"].view(n, H, D).copy_(_rotate(s["q"].view(n, H, D), cos, sin, c))
    at = s["slot"].long()
    s["kc"][:, at] = _rotate(s["k"].view(n, G, D), cos, sin, c).half().transpose(0, 1)
    s["vc"][:, at] = s["v"].view(n, G, D).half().transpose(0, 1)
    return s["out"], s["kc"], s["vc"]


def _rotate(x, cos, sin, c):
    r = c["rope_dim"]
    y = x.clone()
    if c["layout"] == PAIRS:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y[..., 0:r:2], y[..., 1:r:2] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        y[..., :r // 2], y[..., r // 2:r] = a * cos - b * sin, a * sin + b * cos
    return y


def _attn_tree(s):
    c = s["case"]
    n, H, G, D, L = c["n"], c["n_head"], c["n_kv"], c["head_dim"], c["len"]
    if own:
        lrs, b = _product(), s["bufs"]
        lrs.attn_tree_dev(_context(), lrs.KvCache(b["kc"], b["vc"], G, L + n, D), b["q"], n, H, L, b["mask"],
                          b["out"], scale=1.0 / math.sqrt(D))
        return s["out"]
    bits = (s["mask"][:, :, None] >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1
    seen = bits.reshape(n, -1)[:, :n].bool()
    seen = torch.cat([torch.ones(n, L, dtype=torch.bool, device=DEV), seen], 1)
    q = s["q"].view(n, G, H // G, D).permute(1, 2, 0, 3).reshape(G, H // G * n, D)
    p = torch.matmul(q, s["kc"].float().transpose(1, 2).contiguous()) * (1.0 / math.sqrt(D))
    p = p.view(G, H // G, n, L + n).masked_fill_(~seen, -math.inf)
    p = torch.exp(p - p.amax(3, keepdim=True))
    p = (p / p.sum(3, keepdim=True)).view(G, H // G * n, L + n)
    o = torch.matmul(p, s["vc"].float()).view(G, H // G, n, D)
    return o.permute(2, 0, 1, 3).reshape(n, H * D)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    k = case["kind"]
    if k == "sample":
        N = case["rows"] * case["vocab"]
        return dict(bytes=4 * N + 12 * case["rows"], flops=N)
    n, H, G, D = case["n"], case["n_head"], case["n_kv"], case["head_dim"]
    if k == "rope":
        return dict(bytes=n * D * (8 * H + 12 * G) + 8 * n + 2 * case["rope_dim"],
                    flops=3 * n * (H + G) * case["rope_dim"])
    P = case["len"] + n
    return dict(bytes=4 * P * G * D + 8 * n * H * D + 4 * n * ((n + 31) // 32), flops=4 * n * H * D * P)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    k = case["kind"]
    if k == "sample":
        return _exact_sample(s, case)
    n, H, G, D = case["n"], case["n_head"], case["n_kv"], case["head_dim"]
    if k == "rope":
        r, half = case["rope_dim"], case["rope_dim"] // 2
        th = np.outer(s["pos"].cpu().numpy().astype(np.float64), s["freq"].cpu().numpy().astype(np.float64))
        i = np.arange(half)
        a, b = (2 * i, 2 * i + 1) if case["layout"] == PAIRS else (i, i + half)

        def turn(x, heads):
            x = x.cpu().numpy().astype(np.float64).reshape(n, heads, D)
            z = (x[:, :, a] + 1j * x[:, :, b]) * np.exp(1j * th)[:, None, :]
            x[:, :, a], x[:, :, b] = z.real, z.imag
            return x

        kc, vc, at = s["kc"].double(), s["vc"].double(), s["slot"].long()
        kc[:, at] = torch.from_numpy(turn(s["k"], G).transpose(1, 0, 2).copy()).to(DEV)
        vc[:, at] = s["v"].double().view(n, G, D).permute(1, 0, 2).contiguous()
        return torch.from_numpy(turn(s["q"], H).reshape(n, H * D)).to(DEV), kc, vc
    P, L = case["len"] + n, case["len"]
    seen = np.ones((n, P), bool)
    seen[:, L:] = _ancestors(_tree(seed, n))
    hide = torch.from_numpy(~seen).to(DEV)
    out = torch.empty(n, H, D, dtype=torch.float64, device=DEV)
    q = s["q"].double().view(n, H, D)
    for h in range(H):
        g = h // (H // G)
        score = (q[:, h] @ s["kc"][g].double().T) / math.sqrt(D)
        out[:, h] = torch.softmax(score.masked_fill(hide, -math.inf), 1) @ s["vc"][g].double()
    return out.view(n, H * D)


def _exact_sample(s, case):
    logits, u = s["logits"].cpu().numpy(), s["u"].cpu().numpy()
    temp, top_p, min_p = np.float64(np.float32(case["temp"])), np.float64(np.float32(case["top_p"])), \
        np.float64(np.float32(case["min_p"]))
    toks, probs = [], []
    for x, r in zip(logits, u):
        order = np.argsort(-x, kind="stable")[:case["top_k"] or None]
        w = np.exp((x[order].astype(np.float64) - np.float64(x[order[0]])) / temp)
        c = np.cumsum(w)
        last = len(w) if top_p >= 1.0 else int(np.argmax(c >= top_p * c[-1])) + 1
        last = max(1, min(last, int((w >= min_p).sum())))
        words = np.sort(order[:last])
        w = np.exp((x[words].astype(np.float64) - np.float64(x[order[0]])) / temp)
        c = np.cumsum(w)
        j = min(int(np.searchsorted(c, np.float64(r) * c[-1], side="right")), last - 1)
        toks.append(words[j])
        probs.append(w[j] / c[-1])
    return torch.tensor(np.array(toks), dtype=torch.int32), torch.tensor(np.array(probs), dtype=torch.float64)
