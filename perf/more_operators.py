"""What the operators of a step with trees of drafted tokens are measured on.

Every sequence of a batch has a tree of candidate tokens: node 0 is its last token, a node's parent comes before it.  One forward
scores all nodes, tokens are sampled at each of them, and the path that they agree with stays.  Each case is one call of one operator:

* ``mask``       from parents to the nodes that each node sees, as bits, and positions (`ops.tree_mask`)
* ``attention``  of the nodes over a paged cache that holds context and nodes (`ops.tree_attention`)
* ``sample``     a token per row of logits: temperature, top-k, top-p, min-p and a given uniform number per row (`ops.sample`)
* ``accept``     the accepted path, and its keys and values moved to their places in all pools (`ops.tree_accept`)

The nodes of sequence b are rows cu_q[b] .. cu_q[b + 1] and the last positions of its kv_lens[b] in the cache.
"""
import math
import random

import numpy as np
import torch

own = False

_BS = 64                   # tokens of a cache block
_VOCAB = 32000


def _named(c, name):
    return dict(c, name=name) if name else c


def _mask(B, nodes, name=None):
    return _named({"op": "mask", "B": B, "nodes": nodes, "ctx": 500}, name)


def _attention(B, nodes, ctx, hq, hkv, D, int8=False, window=0, keep=0, softcap=0.0, sinks=False, name=None):
    return _named({"op": "attention", "B": B, "nodes": nodes, "ctx": ctx, "hq": hq, "hkv": hkv, "D": D, "int8": int8, "window": window,
                   "keep": keep, "softcap": softcap, "sinks": sinks}, name)


def _sample(rows, V, kind, bf16=False, name=None):
    return _named({"op": "sample", "rows": rows, "V": V, "kind": kind, "bf16": bf16}, name)


def _accept(B, nodes, layers, hkv, D, int8=False, name=None):
    return _named({"op": "accept", "B": B, "nodes": nodes, "ctx": 150, "layers": layers, "hkv": hkv, "D": D, "int8": int8}, name)


def listed():
    return [
        # one user's draft tree, and a server's batch of them
        _mask(1, 26, "mask-1"),
        _mask(192, 64, "mask-192"),
        # one user of an 8B model with grouped heads, short context: nothing but latency
        _attention(1, 16, 700, 32, 8, 128, name="tree-1"),
        # 70B, the benchmark's batch of 16 with prompts of 2048, trees of up to 32 nodes, ragged
        _attention(16, 32, 2100, 64, 8, 128, name="tree-batch"),
        # one long document, a wide tree: 512 rows over each key
        _attention(1, 64, 65536, 64, 8, 128, name="tree-long"),
        # a head of its own for every query (7B, batch 32, prompts of 1024), short drafts
        _attention(32, 8, 1080, 32, 32, 128, name="tree-mha"),
        # 8-bit cache, grouped heads
        _attention(16, 13, 3500, 64, 8, 128, int8=True, name="tree-int8"),
        # one user's step: few candidates
        _sample(1, 32000, "top-k", name="sample-1"),
        # a server's batch, every request with its own parameters
        _sample(64, 128256, "mixed", name="sample-64"),
        # a token for every node of a batch of trees, wide vocabulary, no limit on the candidates' number
        _sample(512, 151936, "top-p", name="sample-512"),
        # one user's tree (8B), and a batch of them (70B)
        _accept(1, 16, 32, 8, 128, name="accept-1"),
        _accept(16, 64, 80, 8, 128, name="accept-16"),
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    op = rng.choice(["mask", "attention", "attention", "attention", "sample", "sample", "accept"])
    if op == "mask":
        return _mask(_log(rng, 1, 192), _log(rng, 12, 256))
    if op == "attention":
        D = rng.choice([64, 128, 128, 128, 128, 256])
        group, hkv = rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 8, 12, 16]), rng.choice([1, 2, 4, 5, 8, 8, 16, 32])
        nodes = _log(rng, 1, 200 if rng.random() < 0.2 else 64)
        most = 64 * 65536 * 8 * 128                                           # keys x rows x their size, of the largest listed one
        ctx = _log(rng, 1, max(2, min(65536, most // (nodes * hkv * D))))
        B = _log(rng, 1, max(1, min(64, most // (ctx * nodes * hkv * D), (1 << 30) // (4 * (ctx + nodes) * hkv * D))))
        window = rng.choice([0, 0, 0, 0, 0, _log(rng, 8, 4096)])
        return _attention(B, nodes, ctx, hkv * group, hkv, D, rng.random() < 0.25, window, rng.choice([0, 4]) if window else 0,
                          rng.choice([0.0, 0.0, 0.0, 0.0, 30.0]), rng.random() < 0.15)
    if op == "sample":
        V = _log(rng, 500, 256000)
        return _sample(_log(rng, 1, max(1, min(512, 512 * 151936 // V))), V,
                       rng.choice(["top-k", "top-p", "min-p", "mixed", "mixed", "none", "flat"]), rng.random() < 0.2)
    hkv, D = rng.choice([1, 2, 4, 8, 32]), rng.choice([64, 128, 128, 256])
    B, nodes = _log(rng, 1, 48), _log(rng, 1, 128)
    layers = _log(rng, 1, 80)
    while B * layers * hkv * D * (150 + nodes) > 16 * 80 * 8 * 128 * 214:
        B, layers = max(1, B // 2), max(1, layers * 2 // 3)
    return _accept(B, nodes, layers, hkv, D, rng.random() < 0.25)


# -- inputs ---------------------------------------------------------------------------------------------------------
def _lens(case):
    """(nodes, context) of each sequence: ragged batches."""
    n, c = case["nodes"], case["ctx"]
    return [(n - (5 * b) % (n // 3 + 1), c - (97 * b) % (c // 4 + 1)) for b in range(case["B"])]


def _shape(b, n):
    """(length of the first chain, nodes of it that are accepted, nodes of the branch that are accepted behind them) of sequence b."""
    d = min(n - 1, max(1, n // 3))
    m = min(1 + b % 3, n - 1 - d, d)
    return d, (2 * b + 1) % (d - m + 1), m


def _tree(rnd, b, n):
    """Parents of a tree of n nodes: the likeliest chain first, a branch that leaves it, then alternatives all over, none deeper."""
    d, a, m = _shape(b, n)
    parents = list(range(-1, d))
    depth = list(range(d + 1))
    while len(parents) < n:
        i = len(parents)
        p = (a if i == d + 1 else i - 1) if i <= d + m else rnd.choice([j for j in range(i) if depth[j] < max(d, 1)])
        parents.append(p)
        depth.append(depth[p] + 1)
    return parents


def _trees(case, seed):
    rnd = random.Random(seed)
    return [_tree(rnd, b, n) for b, (n, _) in enumerate(_lens(case))]


def _parameters(g, kind, rows):
    """(temperature, top_k, top_p, min_p) per row, as requests come."""
    u = torch.rand(4, rows, generator=g, device="cuda")
    T = 0.6 + 0.6 * u[0]
    k = torch.zeros(rows, dtype=torch.int32, device="cuda")
    p, m = torch.ones(rows, device="cuda"), torch.zeros(rows, device="cuda")
    if kind in ("top-k", "mixed"):
        k = (20 + 60 * u[1]).int()
    if kind in ("top-p", "mixed"):
        p = 0.8 + 0.18 * u[2]
    if kind in ("min-p", "mixed"):
        m = 0.02 + 0.1 * u[3]
    if kind == "mixed":                                   # some requests are greedy, some do without one limit or another
        r = torch.arange(rows, device="cuda")
        T = torch.where(r % 8 == 5, 0.0, T)
        k = torch.where(r % 4 == 2, 0, k)
        p = torch.where(r % 4 == 3, 1.0, p)
        m = torch.where(r % 4 != 1, 0.0, m)
    if kind == "flat":                                    # high temperature, and many candidates stay
        T, k, p = 1.5 + u[0], (3000 * u[1]).int() * (u[3] < 0.5), 0.9 + 0.1 * u[2]
    return T, k, p, m


def _logits(g, rows, V, bf16):
    """A wide bulk and a few tokens above it, fewer the higher."""
    x = 2.2 * torch.randn(rows, V, generator=g, device="cuda")
    few = min(V, 64)
    at = (torch.randint(0, V, (rows, 1), generator=g, device="cuda") + torch.arange(few, device="cuda") * (V // few)) % V
    x.scatter_(1, at, 14.0 - 2.0 * torch.log1p(torch.arange(few, device="cuda", dtype=torch.float32)) + torch.randn(rows, few, generator=g, device="cuda"))
    return x.bfloat16() if bf16 else x


def _pool(g, blocks, hkv, D, int8):
    x = torch.randn(blocks, hkv, _BS, D, generator=g, device="cuda", dtype=torch.bfloat16)
    if not int8:
        return x, None
    top = x.abs().amax(-1).float().clamp_min(1e-6) / 127
    return (x.float() / top[..., None]).round().to(torch.int8), top


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = dict(case)
    if case["op"] == "sample":
        s["logits"] = _logits(g, case["rows"], case["V"], case["bf16"])
        s["T"], s["k"], s["p"], s["m"] = _parameters(g, case["kind"], case["rows"])
        s["u"] = torch.rand(case["rows"], generator=g, device="cuda")
        return s
    lens = _lens(case)
    trees = _trees(case, seed)
    s["cu_q"] = [0]
    for n, _ in lens:
        s["cu_q"].append(s["cu_q"][-1] + n)
    s["kv_lens"] = [n + c for n, c in lens]
    s["parents"] = torch.tensor([p for t in trees for p in t], dtype=torch.int32, device="cuda")
    s["cu_dev"] = torch.tensor(s["cu_q"], dtype=torch.int32, device="cuda")
    s["kv_dev"] = torch.tensor(s["kv_lens"], dtype=torch.int32, device="cuda")
    need = [-(-n // _BS) for n in s["kv_lens"]]
    order = torch.randperm(sum(need), generator=g, device="cuda").int()
    s["table"] = torch.zeros(len(need), max(need), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        s["table"][b, :n] = order[at:at + n]
        at += n
    T = s["cu_q"][-1]
    if case["op"] == "attention":
        hq, hkv, D = case["hq"], case["hkv"], case["D"]
        s["q"] = (1.5 * torch.randn(T, hq, D, generator=g, device="cuda")).bfloat16()
        s["kc"], s["ks"] = _pool(g, at, hkv, D, case["int8"])
        s["vc"], s["vs"] = _pool(g, at, hkv, D, case["int8"])
        s["sink"] = torch.randn(hq, generator=g, device="cuda") if case["sinks"] else None
        s["mask"], s["pos"] = _plain_mask(s)
    if case["op"] == "accept":
        for name in "kv":                                    # one allocation, a pool per layer of it
            x, scale = _pool(g, case["layers"] * at, case["hkv"], case["D"], case["int8"])
            s[name + "c"] = x.view(case["layers"], at, *x.shape[1:])
            s[name + "s"] = None if scale is None else scale.view(case["layers"], at, *scale.shape[1:])
        s["pools"] = [None if s[x] is None else list(s[x].unbind()) for x in ("kc", "vc", "ks", "vs")]
        tokens, sampled = _drafts(case, seed, trees)
        s["tokens"], s["sampled"] = torch.tensor(tokens, device="cuda"), torch.tensor(sampled, device="cuda")
    if own:                                                  # the batch that a program's step has made for all of its layers, and its pools
        from xfastertransformer_b200 import ops
        from xfastertransformer_b200.models.decoder import Batch
        if "pools" in s:
            s["handle"] = ops.cache_pools(*s["pools"])
        s["batch"] = Batch(ids=s.get("tokens"), positions=s.get("pos"), slots=None, cu_q=s["cu_q"], kv_lens=s["kv_lens"],
                           block_table=s["table"], cu_q_dev=s["cu_dev"], kv_lens_dev=s["kv_dev"], max_q=max(n for n, _ in lens),
                           max_kv=max(s["kv_lens"]))
    return s


def _drafts(case, seed, trees):
    """Drafted tokens, and sampled ones that agree with a part of the first chain and the branch behind it."""
    rnd = random.Random(seed + 1)
    tokens, sampled = [], []
    for b, t in enumerate(trees):
        mine = rnd.sample(range(_VOCAB // 2), len(t))
        says = [rnd.randrange(_VOCAB // 2, _VOCAB) for _ in t]
        d, a, m = _shape(b, len(t))
        path = list(range(a + 1)) + list(range(d + 1, d + m + 1))
        for i, j in zip(path, path[1:]):
            says[i] = mine[j]
        tokens += mine
        sampled += says
    return tokens, sampled


# -- plain form -----------------------------------------------------------------------------------------------------
def _sequences(s):
    """(sequence, index in its tree) of each row."""
    row = torch.arange(s["cu_q"][-1], device="cuda")
    seq = torch.searchsorted(s["cu_dev"][1:].contiguous(), row, right=True)
    return seq, row - s["cu_dev"].long()[seq]


def _plain_mask(s):
    seq, i = _sequences(s)
    most = max(b - a for a, b in zip(s["cu_q"], s["cu_q"][1:]))
    sees = torch.zeros(i.numel(), -(-most // 64) * 64, dtype=torch.bool, device="cuda")
    first = s["cu_dev"].long()[seq]
    at, live = i, torch.ones_like(i, dtype=torch.bool)
    row = torch.arange(i.numel(), device="cuda")
    depth = torch.full_like(i, -1)
    for _ in range(most):
        sees[row, at] |= live
        depth += live
        up = s["parents"].long()[first + at]
        live = live & (up >= 0)
        at = torch.where(live, up, at)
    bits = sees.view(i.numel(), -1, 64).long() << torch.arange(64, device="cuda")
    n = (s["cu_dev"][1:] - s["cu_dev"][:-1]).long()[seq]
    return bits.sum(-1), (s["kv_dev"].long()[seq] - n + depth).int()


def _rows(cache, scale, table, n):
    """[n, heads, D] in fp32: the first n positions of a sequence."""
    x = cache[table[:-(-n // _BS)].long()].float()
    if scale is not None:
        x = x * scale[table[:-(-n // _BS)].long()][..., None]
    return x.transpose(1, 2).reshape(-1, x.shape[1], x.shape[3])[:n]


def _plain_attention(s):
    D, hkv = s["D"], s["hkv"]
    out = torch.empty_like(s["q"])
    for b, n in enumerate(s["kv_lens"]):
        a, z = s["cu_q"][b], s["cu_q"][b + 1]
        k, v = (_rows(s[x + "c"], s[x + "s"], s["table"][b], n) for x in "kv")
        q = s["q"][a:z].float().view(z - a, hkv, -1, D)
        x = torch.einsum("nhgd,khd->hgnk", q, k) * D ** -0.5
        if s["softcap"]:
            x = s["softcap"] * torch.tanh(x / s["softcap"])
        bits = (s["mask"][a:z, :, None] >> torch.arange(64, device="cuda") & 1).view(z - a, -1)[:, :z - a].bool()
        sees = torch.cat([torch.ones(z - a, n - (z - a), dtype=torch.bool, device="cuda"), bits], 1)
        if s["window"]:
            pos, c = s["pos"][a:z, None], n - (z - a)
            key = torch.cat([torch.arange(c, device="cuda", dtype=torch.int32), s["pos"][a:z]])
            sees &= (pos - key < s["window"]) | (key < s["keep"])
        x = x.masked_fill(~sees, -math.inf)
        top = x.amax(-1, keepdim=True).clamp_min(-1e30)
        e = torch.exp(x - top)
        total = e.sum(-1, keepdim=True)
        if s["sink"] is not None:
            total = total + torch.exp(s["sink"].view(hkv, -1, 1, 1) - top)
        o = torch.einsum("hgnk,khd->nhgd", e, v) / total.clamp_min(1e-30).permute(2, 0, 1, 3)
        out[a:z] = o.reshape(z - a, -1, D).to(out.dtype)
    return out


def _plain_sample(s):
    x, at = torch.sort(s["logits"].double(), dim=1, descending=True, stable=True)
    T = s["T"].double()[:, None]
    w = torch.exp((x - x[:, :1]) / torch.where(T > 0, T, 1.0))
    V = w.shape[1]
    j = torch.arange(V, device="cuda")
    k = torch.where((s["k"] > 0) & (s["k"] < V), s["k"].long(), V)[:, None]
    w = torch.where(j < k, w, 0.0)
    before = torch.cumsum(w, 1) - w
    p = s["p"].double()[:, None]
    keep = (p >= 1) | (before < p * w.sum(1, keepdim=True)) | (j == 0)
    keep &= (w >= s["m"].double()[:, None]) | (j == 0)
    c = torch.cumsum(torch.where(keep, w, 0.0), 1)
    pick = (c <= s["u"].double().clamp(0, 1 - 2.0 ** -24)[:, None] * c[:, -1:]).sum(1).clamp_max(V - 1)
    return at.gather(1, torch.where(s["T"] > 0, pick, 0)[:, None])[:, 0]


def _plain_accept(s):
    seq, i = _sequences(s)
    B, most = s["B"], max(b - a for a, b in zip(s["cu_q"], s["cu_q"][1:]))
    first, n = s["cu_dev"].long()[:-1], (s["cu_dev"][1:] - s["cu_dev"][:-1]).long()
    pad = torch.full((B, most), -2, dtype=torch.long, device="cuda")
    parents, tokens, says = pad.clone(), pad.clone(), pad.clone()
    parents[seq, i], tokens[seq, i], says[seq, i] = s["parents"].long(), s["tokens"], s["sampled"]
    emitted, path = torch.full_like(pad, -1), torch.full_like(pad, -1)
    at, live = torch.zeros_like(n), n > 0
    for j in range(most):
        said = says.gather(1, at[:, None])
        path[:, j] = torch.where(live, at, -1)
        emitted[:, j] = torch.where(live, said[:, 0], -1)
        fits = (parents == at[:, None]) & (tokens == said)
        live = live & fits.any(1)
        at = torch.where(live, fits.long().argmax(1), at)
    count = (path >= 0).sum(1)
    j = torch.arange(most, device="cuda")[None]
    to = torch.where(path >= 0, j, 0)
    c = (s["kv_dev"].long() - n)[:, None]
    src, dst = c + torch.where(path >= 0, path, 0), c + to
    table = s["table"].long()
    sb, db = table.gather(1, src // _BS), table.gather(1, dst // _BS)
    for pools in s["pools"]:
        for x in pools or []:
            x[db, :, dst % _BS] = x[sb, :, src % _BS]
    return emitted, path.int(), count.int(), s["kc"], s["vc"], s["ks"], s["vs"]


def _plain(s):
    return {"mask": _plain_mask, "attention": _plain_attention, "sample": _plain_sample, "accept": _plain_accept}[s["op"]](s)


# -- the framework's ------------------------------------------------------------------------------------------------
def _calls(s):
    from xfastertransformer_b200 import ops
    if s["op"] == "sample":
        return ops.sample(s["logits"], s["T"], s["k"], s["p"], s["m"], s["u"])
    if s["op"] == "mask":
        return ops.tree_mask(s["parents"], s["cu_q"], s["kv_lens"], meta=s["batch"])
    if s["op"] == "attention":
        return ops.tree_attention(s["q"], s["kc"], s["vc"], s["table"], s["cu_q"], s["kv_lens"], s["mask"], s["D"] ** -0.5, ks=s["ks"],
                                  vs=s["vs"], meta=s["batch"], softcap=s["softcap"], window=s["window"], keep_first=s["keep"],
                                  sinks=s["sink"], positions=s["pos"])
    emitted, path, count = ops.tree_accept(s["tokens"], s["parents"], s["sampled"], s["cu_q"], s["kv_lens"], s["table"], s["handle"],
                                           meta=s["batch"])
    return emitted, path, count, s["kc"], s["vc"], s["ks"], s["vs"]


def run(state):
    return _calls(state) if own else _plain(state)


# -- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["V"]
        return {"bytes": n * (2 if case["bf16"] else 4) + case["rows"] * (20 + 8), "flops": 4.0 * n}
    lens = _lens(case)
    T = sum(n for n, _ in lens)
    words = -(-max(n for n, _ in lens) // 64)
    if case["op"] == "mask":
        return {"bytes": T * (4 + 8 * words + 4) + 8 * len(lens), "flops": 2.0 * T}
    hkv, D = case["hkv"], case["D"]
    row = hkv * (D + 4) if case["int8"] else hkv * D * 2                       # a key, or a value, of all heads
    if case["op"] == "attention":
        seen = [min(c, case["window"] + case["keep"]) if case["window"] else c for _, c in lens]
        return {"bytes": sum((n + c) * 2 * row for (n, _), c in zip(lens, seen)) + T * (case["hq"] * D * 4 + 8 * words),
                "flops": sum(4.0 * D * case["hq"] * n * (c + 1) for (n, _), c in zip(lens, seen))}
    moved = sum(_shape(b, n)[2] for b, (n, _) in enumerate(lens))
    return {"bytes": moved * case["layers"] * 2 * row * 2 + T * 20 + len(lens) * 12 * max(n for n, _ in lens), "flops": 1.0 * T}


# -- in 64 bits -----------------------------------------------------------------------------------------------------
def _ancestors(tree, i):
    line = []
    while i >= 0:
        line.append(i)
        i = tree[i]
    return line


def _exact_mask(case, trees):
    words = -(-max(len(t) for t in trees) // 64)
    mask, pos = [], []
    for t, (_, c) in zip(trees, _lens(case)):
        for i in range(len(t)):
            line = _ancestors(t, i)
            bits = [sum(1 << j % 64 for j in line if j // 64 == w) for w in range(words)]
            mask.append([x - (1 << 64) if x >> 63 else x for x in bits])
            pos.append(c + len(line) - 1)
    return torch.tensor(mask, device="cuda"), torch.tensor(pos, dtype=torch.int32, device="cuda")


def _exact_attention(case, s, trees):
    D, hkv = case["D"], case["hkv"]
    group = case["hq"] // hkv
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, (t, (n, c)) in enumerate(zip(trees, _lens(case))):
        lines = [_ancestors(t, i) for i in range(n)]
        hidden = np.zeros((n, c + n), dtype=bool)
        hidden[:, c:] = True
        for i, line in enumerate(lines):
            hidden[i, [c + j for j in line]] = False
            if case["window"]:
                at = np.concatenate([np.arange(c), c - 1 + np.array([len(x) for x in lines])])
                hidden[i] |= (at[c + i] - at >= case["window"]) & (at >= case["keep"])
        hidden = torch.from_numpy(hidden).cuda()
        where = torch.arange(c + n, device="cuda")
        blk, off = s["table"][b].long()[where // _BS], where % _BS
        for h in range(hkv):
            k, v = s["kc"][blk, h, off].double(), s["vc"][blk, h, off].double()
            if case["int8"]:
                k, v = k * s["ks"][blk, h, off].double()[:, None], v * s["vs"][blk, h, off].double()[:, None]
            q = s["q"][s["cu_q"][b]:s["cu_q"][b + 1], h * group:(h + 1) * group].double().reshape(n * group, D)
            x = torch.matmul(q, k.T) / math.sqrt(D)
            if case["softcap"]:
                x = torch.tanh(x / case["softcap"]) * case["softcap"]
            x[hidden.repeat_interleave(group, 0)] = -math.inf
            if case["sinks"]:
                x = torch.cat([x, s["sink"][h * group:(h + 1) * group].double().repeat(n)[:, None]], 1)
            w = torch.exp(x - torch.logsumexp(x, 1, keepdim=True))[:, :c + n]
            out[s["cu_q"][b]:s["cu_q"][b + 1], h * group:(h + 1) * group] = torch.matmul(w, v).view(n, group, D)
    return out


def _exact_sample(s):
    out = []
    host = {n: s[n].double().cpu().numpy() for n in "Tkpmu"}
    for r, row in enumerate(s["logits"].float().cpu().numpy()):
        order = np.argsort(-row, kind="stable")
        T = host["T"][r]
        if not T > 0:
            out.append(int(order[0]))
            continue
        if 0 < host["k"][r] < row.size:
            order = order[:int(host["k"][r])]
        z = row[order].astype(np.float64)
        w = np.exp((z - z[0]) / T)
        total = np.cumsum(w.astype(np.longdouble))
        left = w.size
        if host["p"][r] < 1:                                              # elements with less than the share in front of them
            left = 1 + int(np.searchsorted(total[:-1], np.longdouble(host["p"][r]) * total[-1], side="left"))
        left = min(left, max(1, int((w >= host["m"][r]).sum())))
        u = min(max(host["u"][r], 0.0), 1 - 2.0 ** -24)
        out.append(int(order[np.searchsorted(total[:left], np.longdouble(u) * total[left - 1], side="right")]))
    return torch.tensor(out, device="cuda")


def _exact_accept(case, s, trees):
    most = max(len(t) for t in trees)
    emitted, path, count = [], [], []
    tokens, says = s["tokens"].tolist(), s["sampled"].tolist()
    table = s["table"].tolist()
    moves = []
    for b, (t, (n, c)) in enumerate(zip(trees, _lens(case))):
        base, line = s["cu_q"][b], [0]
        while True:
            fits = [i for i in range(n) if t[i] == line[-1] and tokens[base + i] == says[base + line[-1]]]
            if not fits:
                break
            line.append(fits[0])
        emitted.append([says[base + i] for i in line] + [-1] * (most - len(line)))
        path.append(line + [-1] * (most - len(line)))
        count.append(len(line))
        moves += [(table[b][(c + i) // _BS], (c + i) % _BS, table[b][(c + j) // _BS], (c + j) % _BS) for j, i in enumerate(line) if i != j]
    for pools in (s["kc"], s["vc"], s["ks"], s["vs"]):
        if pools is not None:
            for sb, so, db, do in moves:
                pools[:, db, :, do] = pools[:, sb, :, so]
    dev = {"device": "cuda"}
    return (torch.tensor(emitted, **dev), torch.tensor(path, dtype=torch.int32, **dev), torch.tensor(count, dtype=torch.int32, **dev),
            s["kc"], s["vc"], s["ks"], s["vs"])


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "sample":
        return _exact_sample(s)
    trees = _trees(case, seed)
    if case["op"] == "mask":
        return _exact_mask(case, trees)
    return _exact_attention(case, s, trees) if case["op"] == "attention" else _exact_accept(case, s, trees)
