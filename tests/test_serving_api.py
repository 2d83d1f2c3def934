"""Host-side refusals of the serving operators, in Python and at the C entry points (no device work), and the plain
forms the GPU tests compare against checked on cases worked out by hand."""

import ctypes
import math

import numpy as np
import pytest
import torch

import tree_sparse_flashattn as tsf
from oracle import serving_oracle as so
from tests import serving_util as su
from tsfa import _lib

BF = torch.bfloat16


def _append_args(**change):
    q_lens, kv_lens = [3, 2], [20, 40]
    cache, lists = su.pool(q_lens, kv_lens, 2, 64, BF, 16)
    indices, indptr = su.tables(lists)
    q_indptr, kl = su.lengths(q_lens, kv_lens)
    a = dict(q=torch.zeros(5, 4, 64, dtype=BF), k=torch.zeros(5, 2, 64, dtype=BF), v=torch.zeros(5, 2, 64, dtype=BF),
             kv_cache=cache, kv_indices=indices, positions=torch.arange(5), inv_freq=su.inv_freq(64),
             q_indptr=q_indptr, kv_lens=kl, kv_indptr=indptr)
    a.update(change)
    return a


@pytest.mark.parametrize("change,exc", [
    (dict(q=torch.zeros(5, 256, dtype=BF)), ValueError),
    (dict(k=torch.zeros(4, 2, 64, dtype=BF)), ValueError),                     # tokens
    (dict(v=torch.zeros(5, 3, 64, dtype=BF)), ValueError),                     # heads
    (dict(k=torch.zeros(5, 2, 32, dtype=BF)), ValueError),                     # head_dim
    (dict(kv_layout="NDH"), ValueError),
    (dict(kv_cache=torch.zeros(4, 1, 16, 2, 64, dtype=BF)), ValueError),       # no V slot
    (dict(kv_cache=torch.zeros(4, 2, 8, 2, 64, dtype=BF)), NotImplementedError),
    (dict(kv_cache=torch.zeros(4, 2, 48, 2, 64, dtype=BF)), NotImplementedError),
    (dict(kv_indices=torch.zeros(5, dtype=torch.int64)), ValueError),
    (dict(kv_indptr=None), ValueError),                                        # a 1-D list is no dense table
    (dict(kv_indptr=torch.zeros(2, dtype=torch.int32)), ValueError),
    (dict(q_indptr=torch.zeros(2, dtype=torch.int32)), ValueError),
    (dict(q_indptr=torch.zeros(3, dtype=torch.int64)), ValueError),
    (dict(kv_lens=torch.zeros(2, dtype=torch.float32)), ValueError),
    (dict(positions=torch.zeros(5)), ValueError),
    (dict(positions=torch.zeros(4, dtype=torch.int64)), ValueError),
    (dict(inv_freq=torch.zeros(32, dtype=torch.float64)), ValueError),
    (dict(attention_scaling=math.inf), ValueError),
    (dict(out=torch.zeros(5, 2, 64, dtype=BF)), ValueError),
    (dict(out=torch.zeros(5, 4, 64)), NotImplementedError),
    (dict(v=torch.zeros(5, 2, 64)), NotImplementedError),                      # dtypes differ
    (dict(), ValueError),                                                      # CPU tensors
])
def test_append_refusals(change, exc):
    with pytest.raises(exc):
        tsf.append_paged_kv(**_append_args(**change))


def _attend_args(**change):
    a = _append_args()
    a = dict(q=a["q"], kv_cache=a["kv_cache"], kv_indices=a["kv_indices"], tree_mask=su.tree_masks([3, 2]),
             q_indptr=a["q_indptr"], kv_lens=a["kv_lens"], kv_indptr=a["kv_indptr"])
    a.update(change)
    return a


@pytest.mark.parametrize("change,exc", [
    (dict(q=torch.zeros(5, 4, 128, dtype=BF)), ValueError),
    (dict(q=torch.zeros(5, 3, 64, dtype=BF)), ValueError),                     # 3 query heads on 2 kv heads
    (dict(tree_mask=torch.zeros(3, 4)), ValueError),
    (dict(tree_mask=torch.zeros(3, 4, 4)), ValueError),                        # 3 trees for 2 sequences
    (dict(tree_mask=torch.zeros(0, 0)), ValueError),
    (dict(kv_layout="HDN"), ValueError),
    (dict(kv_indptr=None), ValueError),
    (dict(kv_lens=torch.zeros(3, dtype=torch.int32)), ValueError),
    (dict(q=torch.zeros(5, 4, 64)), NotImplementedError),
    (dict(out=torch.zeros(4, 4, 64, dtype=BF)), ValueError),
    (dict(), ValueError),                                                      # CPU tensors
])
def test_attention_refusals(change, exc):
    with pytest.raises(exc):
        tsf.tree_sparse_attention_fwd_paged_varlen(**_attend_args(**change))


@pytest.mark.parametrize("change,exc", [
    (dict(logits=torch.zeros(2, 30)), ValueError),
    (dict(scores=torch.zeros(2, 4)), ValueError),
    (dict(scores=torch.zeros(2, 3, dtype=BF)), ValueError),
    (dict(k=0), ValueError),
    (dict(k=91), ValueError),                                                  # W * V = 90 continuations
    (dict(logits=torch.zeros(2, 3, 30, dtype=torch.float64)), NotImplementedError),
    (dict(), ValueError),                                                      # CPU tensors
])
def test_select_refusals(change, exc):
    a = dict(logits=torch.zeros(2, 3, 30), scores=torch.zeros(2, 3), k=4)
    a.update(change)
    with pytest.raises(exc):
        tsf.beam_select(a["logits"], a["scores"], a["k"])


# ------------------------------------------------------------- C entry points
OK = dict(batch=2, total_q=5, num_heads=4, num_kv_heads=2, head_dim=64, dtype=_lib.TSFA_DTYPE_BF16)
FAKE = 0x2000  # aligned, never dereferenced: every call here is refused on the host


def _c_attend(mask=FAKE, mask_n=8, n_indices=8, pt_stride=4, pt_width=4, indptr=None, n_pages=8, page_size=16,
              q_strides=(256, 64, 1), cache_strides=(4096, 2048, 128, 64, 1), o_strides=(256, 64, 1), scale=0.1, q=FAKE,
              ws=FAKE, ws_bytes=0, **kw):
    a = dict(OK)
    a.update(kw)
    arr = _lib.i64_array
    return _lib.load().tsfa_fwd_paged_varlen(
        q, FAKE, FAKE, None, mask, 64, 8, mask_n, FAKE, FAKE, indptr, FAKE, n_indices, pt_stride, pt_width, n_pages,
        page_size, arr(q_strides), arr(cache_strides), arr(o_strides), scale, *a.values(), ws, ws_bytes, None)


@pytest.mark.parametrize("kw,status", [
    (dict(num_heads=5), _lib.TSFA_ERR_INVALID_ARGUMENT),
    (dict(batch=-1), _lib.TSFA_ERR_INVALID_ARGUMENT),
    (dict(dtype=_lib.TSFA_DTYPE_FP32), _lib.TSFA_ERR_UNSUPPORTED),
    (dict(head_dim=256), _lib.TSFA_ERR_UNSUPPORTED),
    (dict(num_heads=1024), _lib.TSFA_ERR_UNSUPPORTED),                # 512 heads per kv head
    (dict(total_q=1 << 30), _lib.TSFA_ERR_UNSUPPORTED),
    (dict(scale=math.nan), _lib.TSFA_ERR_INVALID_ARGUMENT),
    (dict(scale=math.inf), _lib.TSFA_ERR_INVALID_ARGUMENT),
    (dict(mask_n=0), _lib.TSFA_ERR_INVALID_ARGUMENT),
    (dict(page_size=8), _lib.TSFA_ERR_UNSUPPORTED),
    (dict(page_size=24), _lib.TSFA_ERR_UNSUPPORTED),
    (dict(n_pages=0), _lib.TSFA_ERR_INVALID_ARGUMENT),
    (dict(n_indices=7), _lib.TSFA_ERR_INVALID_ARGUMENT),              # two lists of four
    (dict(pt_stride=-1), _lib.TSFA_ERR_INVALID_ARGUMENT),
    (dict(q_strides=(256, 64, 2)), _lib.TSFA_ERR_UNSUPPORTED),
    (dict(o_strides=(260, 64, 1)), _lib.TSFA_ERR_UNSUPPORTED),
    (dict(cache_strides=(4096, 2048, 130, 64, 1)), _lib.TSFA_ERR_UNSUPPORTED),
    (dict(cache_strides=(4096, 2048, -128, 64, 1)), _lib.TSFA_ERR_UNSUPPORTED),
    (dict(q=None), _lib.TSFA_ERR_INVALID_ARGUMENT),
    (dict(q=FAKE + 2), _lib.TSFA_ERR_UNSUPPORTED),
    (dict(total_q=0), _lib.TSFA_OK),                                  # nothing to do
    (dict(batch=0), _lib.TSFA_OK),
])
def test_c_attention_checks(kw, status):
    assert _c_attend(**kw) == status


def _c_append(strides=(512, 64, 1) * 4, cache_strides=(4096, 2048, 128, 64, 1), rot=64, freq=FAKE, n_indices=8,
              page_size=16, cache=FAKE, **kw):
    a = dict(OK)
    a.update(kw)
    return _lib.load().tsfa_append_paged_kv(
        FAKE, FAKE, FAKE, FAKE, cache, FAKE, 1, freq, rot, 0, 1.0, FAKE, FAKE, None, FAKE, n_indices, 4, 4, 8,
        page_size, _lib.i64_array(strides), _lib.i64_array(cache_strides), *a.values(), None)


@pytest.mark.parametrize("kw,status", [
    (dict(rot=80), _lib.TSFA_ERR_INVALID_ARGUMENT),                   # above head_dim
    (dict(rot=24), _lib.TSFA_ERR_UNSUPPORTED),
    (dict(head_dim=72), _lib.TSFA_ERR_UNSUPPORTED),
    (dict(head_dim=512), _lib.TSFA_ERR_UNSUPPORTED),
    (dict(dtype=_lib.TSFA_DTYPE_FP32), _lib.TSFA_ERR_UNSUPPORTED),
    (dict(num_kv_heads=0), _lib.TSFA_ERR_INVALID_ARGUMENT),
    (dict(strides=(512, 64, 1) * 3 + (512, 60, 1)), _lib.TSFA_ERR_UNSUPPORTED),
    (dict(cache_strides=(4096, 2048, 128, 64, 2)), _lib.TSFA_ERR_UNSUPPORTED),
    (dict(n_indices=5), _lib.TSFA_ERR_INVALID_ARGUMENT),
    (dict(page_size=12), _lib.TSFA_ERR_UNSUPPORTED),
    (dict(freq=None), _lib.TSFA_ERR_INVALID_ARGUMENT),
    (dict(cache=None), _lib.TSFA_ERR_INVALID_ARGUMENT),
    (dict(cache=FAKE + 8), _lib.TSFA_ERR_UNSUPPORTED),
    (dict(total_q=0), _lib.TSFA_OK),
])
def test_c_append_checks(kw, status):
    assert _c_append(**kw) == status


@pytest.mark.parametrize("kw,status", [
    (dict(k=65), _lib.TSFA_ERR_UNSUPPORTED),
    (dict(k=0), _lib.TSFA_ERR_INVALID_ARGUMENT),
    (dict(beams=300), _lib.TSFA_ERR_UNSUPPORTED),
    (dict(beams=2, vocab=3, k=7), _lib.TSFA_ERR_INVALID_ARGUMENT),
    (dict(vocab=1 << 30), _lib.TSFA_ERR_UNSUPPORTED),
    (dict(batch=1 << 30), _lib.TSFA_ERR_UNSUPPORTED),                 # batch * k rows of states
    (dict(dtype=7), _lib.TSFA_ERR_UNSUPPORTED),
    (dict(n_states=9), _lib.TSFA_ERR_UNSUPPORTED),
    (dict(n_states=-1), _lib.TSFA_ERR_INVALID_ARGUMENT),
    (dict(logits=None), _lib.TSFA_ERR_INVALID_ARGUMENT),
    (dict(), _lib.TSFA_ERR_WORKSPACE),                                # no workspace given
    (dict(batch=0), _lib.TSFA_OK),
])
def test_c_select_checks(kw, status):
    a = dict(logits=FAKE, batch=2, beams=4, vocab=1000, k=5, dtype=1, n_states=0)
    a.update(kw)
    none = (ctypes.c_void_p * 1)()
    st = _lib.load().tsfa_beam_select(a["logits"], 4000, 1000, FAKE, 4, 1, a["batch"], a["beams"], a["vocab"], a["k"],
                                      a["dtype"], FAKE, FAKE, FAKE, none, none, _lib.i64_array([0]), a["n_states"],
                                      None, 0, None)
    assert st == status


def test_select_workspace_is_zero_for_refused_shapes():
    lib = _lib.load()
    assert lib.tsfa_beam_select_workspace_bytes(2, 4, 1000, 5) > 0
    assert lib.tsfa_beam_select_workspace_bytes(2, 4, 1000, 65) == 0


# ------------------------------------------------------------ the plain forms
def test_plain_select_by_hand():
    x = torch.log(torch.tensor([[[1.0, 2.0, 1.0], [6.0, 1.0, 1.0]]]))
    c = torch.log(torch.tensor([[0.5, 0.5]]))
    # probabilities: beam 0 .125 .25 .125, beam 1 .375 .0625 .0625
    tokens, parents, best = so.beam_select(x, c, 4)
    assert tokens.tolist() == [[0, 1, 0, 2]] and parents.tolist() == [[1, 0, 0, 0]]
    np.testing.assert_allclose(np.exp(best), [[0.375, 0.25, 0.125, 0.125]], rtol=1e-6)


def test_plain_rotation_by_hand():
    x = torch.tensor([[[1.0, 0.0, 5.0, 0.0]]])
    quarter = torch.tensor([math.pi / 2])
    out, _ = so.rotate(x, torch.tensor([1]), quarter, interleaved=True)
    np.testing.assert_allclose(out[0, 0].numpy(), [0, 1, 5, 0], atol=1e-6)
    out, _ = so.rotate(x, torch.tensor([1]), torch.tensor([math.pi / 2, 0.0]), interleaved=False)
    np.testing.assert_allclose(out[0, 0].numpy(), [-5, 0, 1, 0], atol=1e-6)


def test_plain_attention_against_the_dense_oracle():
    from oracle.attn_oracle import dense_mask_attention

    g = torch.Generator().manual_seed(0)
    q_lens, kv_lens = [6, 3], [20, 3]
    cache, lists = su.pool(q_lens, kv_lens, 2, 16, torch.float32, 16)
    q = torch.randn(9, 4, 16, generator=g)
    masks = su.tree_masks(q_lens)
    o, _, _, _ = so.varlen_attention(q, cache, lists, masks, q_lens, kv_lens)
    at = 0
    for b, (m, n) in enumerate(zip(q_lens, kv_lens)):
        k, v = so.paged_kv(cache, lists[b], n, "NHD")
        ref = dense_mask_attention(q[at:at + m].transpose(0, 1)[None], k.transpose(0, 1)[None].float(),
                                   v.transpose(0, 1)[None].float(), masks[b, :m, :m], n - m)
        assert float((o[at:at + m] - ref[0].transpose(0, 1)).abs().max()) < 1e-5
        at += m
