"""Inputs shared by the tests of the serving operators."""

from __future__ import annotations

import numpy as np
import torch

from tsfa import trees


def pool(q_lens, kv_lens, hkv, d, dtype, page, layout="NHD", seed=0, spare=2, stale=None, width=None):
    """A page pool on the CPU with scattered pages: (cache, lists).  Rows no sequence owns hold ``stale`` if given."""
    g = torch.Generator().manual_seed(seed)
    counts = [-(-n // page) for n in kv_lens]
    total = sum(counts) + spare
    shape = (total, 2, page, hkv, d) if layout == "NHD" else (total, 2, hkv, page, d)
    cache = torch.randn(shape, generator=g).to(dtype)
    order = torch.randperm(total, generator=g).tolist()
    lists, at = [], 0
    for n in counts:
        lists.append(order[at:at + n])
        at += n
    if stale is not None:
        owned = torch.zeros(total, page, dtype=torch.bool)
        for pages, n in zip(lists, kv_lens):
            for j in range(n):
                owned[pages[j // page], j % page] = True
        rows = cache if layout == "NHD" else cache.transpose(2, 3)
        rows.transpose(1, 2)[~owned] = stale
    return cache, lists


def tables(lists, dense=False, fill=0):
    """(kv_indices, kv_indptr) int32 CSR, or a padded dense table and None."""
    if dense:
        width = max([len(x) for x in lists] + [1])
        return torch.tensor([list(x) + [fill] * (width - len(x)) for x in lists], dtype=torch.int32), None
    flat = [p for x in lists for p in x] or [0]
    return (torch.tensor(flat, dtype=torch.int32),
            torch.tensor(np.concatenate([[0], np.cumsum([len(x) for x in lists])]), dtype=torch.int32))


def lengths(q_lens, kv_lens):
    return (torch.tensor(np.concatenate([[0], np.cumsum(q_lens)]), dtype=torch.int32),
            torch.tensor(kv_lens, dtype=torch.int32))


def tree_masks(q_lens, seed=0, t=None):
    """bool [B, T, T]: a random tree of q_lens[b] tokens in each upper left corner."""
    t = max(q_lens) if t is None else t
    out = np.zeros((len(q_lens), t, t), dtype=bool)
    for b, m in enumerate(q_lens):
        if m:
            out[b, :m, :m] = trees.ancestor_mask(trees.random_parents(m, np.random.default_rng([seed, b])))
    return torch.from_numpy(out)


def inv_freq(rot, base=10000.0):
    half = rot // 2
    return (base ** (-torch.arange(half, dtype=torch.float64) / max(half, 1))).float()
