"""Batches with trees of drafted tokens, for the tests of their operators."""
import random

import torch


def parents_of(rnd, n, roots=1):
    """A tree (or a few) of n nodes, every node's parent before it."""
    return [-1 if i < roots else rnd.randrange(-1 if roots > 1 else 0, i) for i in range(n)]


def ancestors(parents, i):
    line = []
    while i >= 0:
        line.append(i)
        i = parents[i]
    return line


def batch(lens, seed, bs=64, roots=1, spare=2):
    """(parents of each tree, flat parents, cu_q, kv_lens, block table) for (nodes, context) of each sequence; blocks in any order."""
    rnd = random.Random(seed)
    trees = [parents_of(rnd, n, roots) for n, _ in lens]
    cu = [0]
    for n, _ in lens:
        cu.append(cu[-1] + n)
    kv = [n + c for n, c in lens]
    need = [-(-n // bs) for n in kv]
    ids = list(range(sum(need) + spare))
    rnd.shuffle(ids)
    table = torch.zeros(len(lens), max(need + [1]) + 1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(ids[at:at + n], dtype=torch.int32)
        at += n
    flat = torch.tensor([p for t in trees for p in t], dtype=torch.int32)
    return trees, flat, cu, kv, table, len(ids)


def caches(g, blocks, hkv, D, bs=64, int8=False):
    """(keys, values, scales of both or None) with something in every slot."""
    if int8:
        kv = [torch.randint(-127, 128, (blocks, hkv, bs, D), generator=g, dtype=torch.int8) for _ in range(2)]
        return (*kv, *(torch.rand(blocks, hkv, bs, generator=g) * 0.015 + 0.005 for _ in range(2)))
    return (*(torch.randn(blocks, hkv, bs, D, generator=g).bfloat16() for _ in range(2)), None, None)
