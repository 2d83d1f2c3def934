"""Plain 64-bit implementations of the serving operators, on the CPU.

beam_select, append_paged_kv and tree_sparse_attention_fwd_paged_varlen of
tree_sparse_flashattn, written from their definitions with loops over
sequences, heads and tokens; nothing here calls the library.
"""

from __future__ import annotations

import math

import numpy as np
import torch


def paged_kv(cache: torch.Tensor, pages, n_keys: int, layout: str):
    """K, V [n_keys, Hkv, D] float64 of one sequence's page list."""
    if n_keys == 0:
        hkv = cache.shape[3] if layout == "NHD" else cache.shape[2]
        return (torch.zeros(0, hkv, cache.shape[4], dtype=torch.float64),) * 2
    rows = [cache[p] if layout == "NHD" else cache[p].transpose(1, 2) for p in pages]  # [2, page, Hkv, D]
    kv = torch.cat(rows, dim=1)[:, :n_keys].double()
    return kv[0], kv[1]


def varlen_attention(q, cache, lists, mask, q_lens, kv_lens, layout="NHD", sm_scale=None):
    """(O [N, Hq, D], lse [N, Hq], weight of |V| [N, Hq, D], largest sum of |q k| scale) in float64.

    lists: page ids of each sequence; mask: bool [B, T, T], [T, T] or None
    (causal).  Rows without a visible key are 0 with lse -inf.  The last two
    results bound rounding errors: sum_j p_j |v_j|, and the largest
    scale * sum_d |q_d k_d|.
    """
    n, hq, d = q.shape
    scale = d ** -0.5 if sm_scale is None else sm_scale
    o = torch.zeros(n, hq, d, dtype=torch.float64)
    lse = torch.full((n, hq), -math.inf, dtype=torch.float64)
    size = torch.zeros_like(o)
    most = 0.0
    at = 0
    for b, (m, kl) in enumerate(zip(q_lens, kv_lens)):
        k, v = paged_kv(cache, lists[b], kl, layout)
        group = hq // k.shape[1] if k.shape[1] else 1
        prefix = max(kl - m, 0)
        for i in range(m):
            seen = list(range(prefix))
            for j in range(m):
                if prefix + j >= kl:
                    break
                if mask is None:
                    visible = j <= i
                else:
                    tree = mask if mask.dim() == 2 else mask[b]
                    visible = i < tree.shape[0] and j < tree.shape[0] and bool(tree[i, j])
                if visible:
                    seen.append(prefix + j)
            if not seen:
                continue
            ks, vs = k[seen], v[seen]
            for h in range(hq):
                x = q[at + i, h].double()
                s = (ks[:, h // group] @ x) * scale
                lse[at + i, h] = torch.logsumexp(s, 0)
                p = torch.softmax(s, 0)
                o[at + i, h] = p @ vs[:, h // group]
                size[at + i, h] = p @ vs[:, h // group].abs()
                most = max(most, float((ks[:, h // group].abs() @ x.abs()).nan_to_num(0, 0, 0).max()) * abs(scale))
        at += m
    return o, lse, size, most


def attention_tolerance(o, size, most, dtype, n_keys):
    """Largest |difference| the kernel's roundings allow, per element.

    u = eps / 2 of the dtype.  O is rounded once (u |O|) and each weight once
    for the product with V (u sum p |v|).  A score is a 32-bit sum of D
    products, D eps32 most off at worst (eps32 = 2^-23: the matrix unit need not
    round to nearest), and exp2 and its argument add 2^-20 relative; a weight's
    relative error counts twice (numerator and normaliser).  The two sums over
    the keys add n eps32 each, and joining partial results 2^-20.
    """
    u, e = torch.finfo(dtype).eps / 2, 2.0 ** -23
    rel = 2 * (o.shape[-1] * e * most + 2.0 ** -20) + 2 * n_keys * e + 2.0 ** -20
    return u * o.abs() + (u + rel) * (1 + u) * size + 1e-30


def rotate(x, positions, inv_freq, interleaved, scaling=1.0):
    """x [N, H, D] float64 with its first 2 * len(inv_freq) elements turned, and sum of |operands| per element."""
    x = x.double()
    out, size = x.clone(), torch.zeros_like(x)
    half = inv_freq.numel()
    for i in range(half):
        a = positions.double() * float(inv_freq[i].double())
        c, s = torch.cos(a)[:, None] * scaling, torch.sin(a)[:, None] * scaling
        i1, i2 = (2 * i, 2 * i + 1) if interleaved else (i, half + i)
        x1, x2 = x[..., i1], x[..., i2]
        out[..., i1], out[..., i2] = x1 * c - x2 * s, x2 * c + x1 * s
        size[..., i1] = size[..., i2] = (x1.abs() + x2.abs()) * abs(scaling)
    return out, size


def append(q, k, v, cache, lists, positions, inv_freq, q_lens, kv_lens, page, layout="NHD", interleaved=False,
           scaling=1.0):
    """(q rotated, its operand sums, cache float64, operand sums of the cache, which cache rows were written).

    Rows of q behind the last sequence come back as they were.
    """
    used = sum(q_lens)
    qr, qs = q.double().clone(), torch.zeros(q.shape, dtype=torch.float64)
    qr[:used], qs[:used] = rotate(q[:used], positions[:used], inv_freq, interleaved, scaling)
    kr, ks = rotate(k[:used], positions[:used], inv_freq, interleaved, scaling)
    new, size = cache.double().clone(), torch.zeros(cache.shape, dtype=torch.float64)
    written = torch.zeros(cache.shape, dtype=torch.bool)
    at = 0
    for b, (m, kl) in enumerate(zip(q_lens, kv_lens)):
        for i in range(m):
            key = kl - m + i
            if key < 0 or key // page >= len(lists[b]):
                continue
            p = int(lists[b][key // page])
            if not 0 <= p < cache.shape[0]:
                continue
            where = (p, slice(None), key % page) if layout == "NHD" else (p, slice(None), slice(None), key % page)
            new[where] = torch.stack((kr[at + i], v[at + i].double()))
            size[where] = torch.stack((ks[at + i], torch.zeros_like(ks[at + i])))
            written[where] = True
        at += m
    return qr, qs, new, size, written


def beam_select(logits, scores, k):
    """(tokens, parents, scores) as int64 / float64 numpy arrays, from the definition."""
    x = logits.double().numpy().copy()
    x[np.isnan(x)] = -math.inf
    batch, beams, vocab = x.shape
    tokens, parents = np.zeros((batch, k), np.int64), np.zeros((batch, k), np.int64)
    best = np.full((batch, k), -math.inf)
    for b in range(batch):
        value = np.full((beams, vocab), -math.inf)
        for w in range(beams):
            c, row = float(scores[b, w]), x[b, w]
            top = row.max()
            if not math.isfinite(c) or top == -math.inf:
                continue
            if top == math.inf:
                hit = row == math.inf
                value[w, hit] = c - math.log(hit.sum())
                continue
            lse = top + math.log(np.exp(row - top).sum())
            value[w] = (c + row) - lse
        flat = value.reshape(-1)
        order = np.lexsort((np.arange(flat.size), -flat))[:k]
        for i, f in enumerate(order):
            if flat[f] == -math.inf:
                break
            tokens[b, i], parents[b, i], best[b, i] = f % vocab, f // vocab, flat[f]
    return tokens, parents, best
