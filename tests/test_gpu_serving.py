"""beam_select, append_paged_kv and tree_sparse_attention_fwd_paged_varlen on the GPU against their plain 64-bit
forms, at the sizes, lengths and masks where they can go wrong, and as the chain a draft step runs them in."""

import numpy as np
import pytest
import torch

import tree_sparse_flashattn as tsf
from oracle import serving_oracle as so
from tests import serving_util as su

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16
NAN = float("nan")


def _dev(*tensors):
    return [None if t is None else t.cuda() for t in tensors]


def _same(a, b):
    """Bit-equal, NaN where NaN."""
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(7.0, 8.0, 9.0), b.nan_to_num(7.0, 8.0, 9.0))


# ------------------------------------------------------------------ attention
def _attend(q_lens, kv_lens, hq=8, hkv=2, d=128, dtype=BF, page=16, layout="NHD", mask="tree", dense=False, seed=0,
            sm_scale=None, pad=0, stale=NAN, edit=None, check=True, room=0):
    """One call against the plain form; returns what was used.  ``room``: entries behind each page list's last page,
    which the lengths do not reach."""
    g = torch.Generator().manual_seed(1000 + seed)
    n = sum(q_lens)
    cache, lists = su.pool(q_lens, kv_lens, hkv, d, dtype, page, layout, seed, stale=stale)
    q = torch.randn(n + pad, hq, d, generator=g).to(dtype)
    tree = None
    if mask == "tree":
        tree = su.tree_masks(q_lens, seed)
    elif mask == "shared":
        tree = su.tree_masks([max(q_lens)], seed)[0]
    if edit is not None:
        edit(q, cache, lists, tree)
    room = min(room, (1 << 22) // len(lists))
    indices, indptr = su.tables([list(x) + [0] * room for x in lists], dense)
    q_indptr, kl = su.lengths(q_lens, kv_lens)
    dq, dc, di, dp, dqi, dkl, dt = _dev(q, cache, indices, indptr, q_indptr, kl, tree)
    out = torch.full_like(dq, NAN)
    got, lse = tsf.tree_sparse_attention_fwd_paged_varlen(dq, dc, di, dt, q_indptr=dqi, kv_lens=dkl, kv_indptr=dp,
                                                          kv_layout=layout, sm_scale=sm_scale, out=out,
                                                          return_lse=True)
    torch.cuda.synchronize()
    assert got is out
    if check:
        ref, rl, size, most = so.varlen_attention(q[:n], cache, lists, tree, q_lens, kv_lens, layout, sm_scale)
        tol = so.attention_tolerance(ref, size, most, dtype, max(kv_lens, default=0))
        o = got[:n].double().cpu()
        bad = ref.isnan() | ref.isinf()
        assert torch.equal(o.isnan(), ref.isnan())
        diff = torch.where(bad, 0.0, (o - ref).abs())
        worst = float((diff / torch.where(bad, 1.0, tol)).max()) if n else 0.0
        print(f"[attend] worst {worst:.3f} of the tolerance", flush=True)
        assert worst <= 1
        gl = lse[:n].double().cpu()
        assert torch.equal(gl == -torch.inf, rl == -torch.inf)
        ok = torch.isfinite(rl)
        bound = (d + max(kv_lens, default=0)) * 2.0 ** -23 * (1 + most) + 2.0 ** -20 * (1 + rl[ok].abs())
        assert bool(((gl[ok] - rl[ok]).abs() <= bound).all())
    assert bool(got[n:].isnan().all())  # rows behind the last sequence: as they were
    return dict(q=dq, cache=dc, indices=di, indptr=dp, q_indptr=dqi, kv_lens=dkl, tree=dt, out=got, lse=lse)


ATTEND = [
    # q lengths, kv lengths, keywords
    ([1], [1], dict()),                                                     # one token alone
    ([1], [700], dict(mask="causal")),
    ([1, 1, 1], [17, 1, 4100], dict(mask="causal", d=64, dtype=FP)),        # decoding, very different lengths
    ([0, 3, 0, 1, 0], [5, 3, 0, 40, 9], dict()),                            # sequences without queries or keys
    ([5, 33, 64], [5, 33 + 15, 64 + 511], dict()),                          # no prefix; odd prefixes
    ([37, 130], [37 + 101, 130 + 16], dict(dtype=FP, layout="HND", page=64)),
    ([20, 7], [420, 39], dict(hq=4, hkv=4, d=64, page=32)),
    ([9, 50], [73, 306], dict(hq=14, hkv=2, d=64, dtype=FP, layout="HND")),  # 7 heads per kv head
    ([12, 3], [900, 33], dict(hq=8, hkv=1, page=256, dense=True)),
    ([40, 11], [340, 75], dict(mask="shared", dense=True)),                  # one tree, cut to each length
    ([100, 31], [100, 531], dict(mask="causal")),                            # prompts, one behind a cached prefix
    ([300], [300 + 7], dict(mask="causal", hq=4, hkv=1, d=64)),
    ([8, 8], [208, 1008], dict(hq=4, hkv=4)),                                # few rows, 32-row tiles
    ([2] * 70, [3 + 13 * i % 200 for i in range(70)], dict(hq=4, hkv=2, d=64, mask="causal")),  # above 64 sequences
    ([600], [650], dict(hq=2, hkv=2, d=64)),                                 # words of a wide tree in several parts
    ([1], [17000], dict(hq=2, hkv=1, d=64, mask="causal")),                  # a long page list
    ([1, 2], [5000, 2300], dict()),                                          # 32-row tiles, many steps
    ([40], [2100], dict(dtype=FP)),                                          # 128-row tiles, many steps
    ([150, 140], [1050, 1640], dict(hq=8, hkv=1)),                           # 256-row tiles, many steps
    ([90], [700], dict(hq=8, hkv=1, d=64, mask="causal", layout="HND")),
    ([1, 3], [300, 40], dict(hq=256, hkv=1, d=64, mask="causal")),           # more heads than a tile has rows
    ([5, 2, 1], [70, 130, 1], dict(hq=71, hkv=1, dtype=FP)),
    ([1 + i % 2 for i in range(1500)], [1 + 7 * i % 50 for i in range(1500)],
     dict(hq=2, hkv=1, d=64, mask="causal", page=32)),                       # many sequences
]


# Lists with room for few keys take tiles of 32 rows where a call is small, lists with room for many 128 or 256.
ROOM = pytest.mark.parametrize("room", [0, 1 << 18], ids=["tight", "roomy"])


@ROOM
@pytest.mark.parametrize("case", ATTEND, ids=[f"a{i}" for i in range(len(ATTEND))])
def test_varlen_attention(case, room):
    q_lens, kv_lens, kw = case
    print(f"[attend] {q_lens} {kv_lens} {kw} room {room}", flush=True)
    # rows of the pool that hold no key are NaN: none may reach a result
    _attend(q_lens, [max(a, b) for a, b in zip(q_lens, kv_lens)], seed=len(q_lens), room=room, **kw)


# kv heads, query heads per kv head, query tokens, keys, batch, head_dim: every workgroup walks many steps in each of
# the three tile shapes; more keys than its table of pages of 16 keys holds; more of a tree than its table of
# visibility words
LONG = [(8, 4, 1, 6000, 16, 128), (8, 4, 30, 5000, 8, 128), (8, 8, 200, 3000, 2, 128), (8, 8, 200, 4000, 4, 128),
        (16, 8, 512, 17000, 1, 64), (16, 4, 30, 17000, 16, 64), (16, 1, 1, 40000, 8, 64), (16, 8, 700, 760, 1, 64),
        (16, 8, 700, 760, 3, 64)]


@pytest.mark.parametrize("case", LONG, ids=[f"l{i}" for i in range(len(LONG))])
def test_varlen_long_runs(case):
    hkv, group, q_len, keys, batch, d = case
    print(f"[attend] {case}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(q_len)
    n = batch * q_len
    q = torch.randn(n, hkv * group, d, generator=g, device="cuda").to(BF)
    kv = torch.randn(batch, 2, hkv, keys, d, generator=g, device="cuda").to(BF)
    mask = su.tree_masks([q_len])[0].cuda()
    lens = dict(q_indptr=torch.arange(batch + 1, dtype=torch.int32, device="cuda") * q_len,
                kv_lens=torch.full((batch,), keys, dtype=torch.int32, device="cuda"))
    outs = []
    for page in (16, 1024):  # each twice: a wait that is missing shows as a difference between runs
        pages = -(-keys // page)
        cache = torch.zeros(batch, 2, hkv, pages * page, d, dtype=BF, device="cuda")
        cache[:, :, :, :keys] = kv
        cache = cache.view(batch, 2, hkv, pages, page, d).permute(0, 3, 1, 2, 4, 5).reshape(-1, 2, hkv, page, d)
        table = torch.arange(batch * pages, dtype=torch.int32, device="cuda").view(batch, pages)
        for _ in range(2):
            outs.append(tsf.tree_sparse_attention_fwd_paged_varlen(q, cache, table, mask, kv_layout="HND", **lens))
        del cache
    torch.cuda.synchronize()
    # the pages' size changes where a run's tables end and nothing else
    for out in outs[1:]:
        assert torch.equal(outs[0], out)
    # sequences and kv heads in 64 bits
    for b in {0, batch // 2, batch - 1}:
        for h in range(hkv) if keys < 10000 else (0, hkv - 1):
            k, v = kv[b, 0, h].double(), kv[b, 1, h].double()
            rows, heads = slice(b * q_len, (b + 1) * q_len), slice(h * group, (h + 1) * group)
            x = q[rows, heads].double().transpose(0, 1).reshape(-1, d)
            score = (x @ k.t()) * d ** -0.5
            most = float((x.abs() @ k.abs().t()).max()) * d ** -0.5
            score = score.view(group, q_len, keys)
            score[:, :, keys - q_len:].masked_fill_(~mask, -torch.inf)
            w = torch.softmax(score, -1).view(-1, keys)
            ref, size = w @ v, w @ v.abs()
            got = outs[0][rows, heads].double().transpose(0, 1).reshape(-1, d)
            assert bool(((got - ref).abs() <= so.attention_tolerance(ref, size, most, BF, keys)).all())


@ROOM
@pytest.mark.parametrize("sm_scale", [0.0, -0.2, 3.0])
def test_varlen_scales(sm_scale, room):
    print(f"[attend] scale {sm_scale} room {room}", flush=True)
    _attend([10, 33], [90, 65], sm_scale=sm_scale, room=room)


@ROOM
def test_varlen_rows_without_keys_are_zero(room):
    print(f"[attend] empty rows room {room}", flush=True)

    def edit(q, cache, lists, tree):
        tree[0, 3] = False
        tree[1, 0] = False

    s = _attend([6, 4], [6, 4], edit=edit, room=room)
    assert bool((s["out"][3] == 0).all()) and bool((s["out"][6] == 0).all())
    # behind a prefix the same rows see it
    _attend([6, 4], [40, 37], edit=edit, room=room)
    _attend([66, 80], [106, 100], edit=edit, room=room)


@ROOM
def test_varlen_non_finite_values_in_masked_places(room):
    print(f"[attend] masked NaN and infinities room {room}", flush=True)
    for dtype in (BF, FP):
        for bad in (NAN, float("inf"), -float("inf")):
            for q_len, kv_len in ((40, 40), (40, 300), (80, 300)):
                def edit(q, cache, lists, tree):
                    # token 7 is seen by itself and its descendants alone
                    key = kv_len - q_len + 7
                    cache[lists[0][key // 16], 0, key % 16, :, 5] = bad
                    cache[lists[0][key // 16], 1, key % 16] = bad
                    tree[0, 8:, 7] = False
                    tree[0, 7, 7] = False
                    tree[0, 20, 7] = bad == bad  # one row sees the infinities

                s = _attend([q_len], [kv_len], dtype=dtype, edit=edit, check=bad != bad, room=room)
                rows = [i for i in range(q_len) if i != 20 or bad != bad]
                assert bool(s["out"][rows].isfinite().all())
                assert not bool(s["out"][20].isfinite().all()) or bad != bad


def test_varlen_masks_of_other_types_and_strides():
    print("[attend] mask types", flush=True)
    s = _attend([21, 40], [121, 300])
    kw = dict(q_indptr=s["q_indptr"], kv_lens=s["kv_lens"], kv_indptr=s["indptr"])
    wide = torch.zeros(2, 50, 57, dtype=torch.bool, device="cuda")
    wide[:, :40, :40] = s["tree"]
    for mask in (s["tree"].int(), s["tree"].half(), s["tree"].transpose(1, 2).contiguous().transpose(1, 2),
                 wide[:, :40, :40]):
        assert torch.equal(tsf.tree_sparse_attention_fwd_paged_varlen(s["q"], s["cache"], s["indices"], mask, **kw),
                           s["out"])
    # a mask smaller than the longest draft: the rest sees and is seen by nothing of the tree
    q_lens, kv_lens = [21, 40], [121, 300]
    small = s["tree"][:, :30, :30].contiguous()
    got = tsf.tree_sparse_attention_fwd_paged_varlen(s["q"], s["cache"], s["indices"], small, **kw)
    cut = torch.zeros_like(s["tree"])
    cut[:, :30, :30] = small
    assert torch.equal(got, tsf.tree_sparse_attention_fwd_paged_varlen(s["q"], s["cache"], s["indices"], cut, **kw))


def test_varlen_strided_queries_and_outputs():
    print("[attend] strides", flush=True)
    s = _attend([5, 30], [50, 95], hq=4, hkv=2, d=64)
    kw = dict(q_indptr=s["q_indptr"], kv_lens=s["kv_lens"], kv_indptr=s["indptr"])
    n = s["q"].shape[0]
    fused = torch.randn(n, 8, 64, device="cuda").to(BF)
    fused[:, 2:6] = s["q"]
    q = fused[:, 2:6]                                           # a view of a fused projection
    heads = s["q"].transpose(0, 1).contiguous().transpose(0, 1)  # [H, N, D] memory
    odd = torch.empty(n, 4, 65, device="cuda", dtype=BF)[..., :64]  # rows no 16-byte load addresses
    odd.copy_(s["q"])
    for x in (q, heads, odd):
        assert torch.equal(tsf.tree_sparse_attention_fwd_paged_varlen(x, s["cache"], s["indices"], s["tree"], **kw),
                           s["out"])
    out = torch.full((n + 2, 4, 65), NAN, device="cuda", dtype=BF)[..., :64]
    tsf.tree_sparse_attention_fwd_paged_varlen(torch.cat([s["q"], s["q"][:2]]), s["cache"], s["indices"], s["tree"],
                                               out=out, **kw)
    assert torch.equal(out[:n], s["out"]) and bool(out[n:].isnan().all())


def test_varlen_equals_the_uniform_paged_forward():
    print("[attend] against the uniform forward", flush=True)
    b, t, p = 3, 24, 100
    s = _attend([t] * b, [p + t] * b)
    meta = tsf.prepare_tree_sparse_metadata_batched(s["tree"], p, 16, 16)
    uniform = tsf.tree_sparse_attention_fwd_paged(s["q"].view(b, t, 8, 128).transpose(1, 2).contiguous(), s["cache"],
                                                  s["indices"], meta, kv_len=p + t, kv_indptr=s["indptr"])
    diff = (uniform.transpose(1, 2).reshape(b * t, 8, 128).double() - s["out"].double()).abs()
    # each rounds O once, and its weights (or split partials) once: |O| <= max |v|
    bound = 4 * torch.finfo(BF).eps / 2 * float(s["cache"].nan_to_num(0).abs().max())
    assert float(diff.max()) <= bound


@ROOM
def test_varlen_device_lengths_out_of_range_read_nothing_outside(room):
    print(f"[attend] lengths and pages out of range room {room}", flush=True)
    s = _attend([5, 12], [50, 95], room=room)
    q, cache = s["q"], s["cache"].nan_to_num(0)
    put = dict(dtype=torch.int32, device="cuda")
    # a list with pages outside the pool, lengths past the list, negative and falling lengths
    wild = s["indices"].clone()
    wild[0], wild[-1] = 1 << 30, -5
    for indices, q_indptr, kv_lens, indptr in (
            (wild, s["q_indptr"], s["kv_lens"], s["indptr"]),
            (s["indices"], s["q_indptr"], torch.tensor([1 << 30, 2000000000], **put), s["indptr"]),
            (s["indices"], s["q_indptr"], torch.tensor([-7, 3], **put), s["indptr"]),
            (s["indices"], torch.tensor([-3, 9, 4], **put), s["kv_lens"], s["indptr"]),
            (s["indices"], torch.tensor([0, 5, 99999], **put), s["kv_lens"], torch.tensor([0, -4, 1 << 29], **put))):
        out = tsf.tree_sparse_attention_fwd_paged_varlen(q, cache, indices, s["tree"], q_indptr=q_indptr,
                                                         kv_lens=kv_lens, kv_indptr=indptr,
                                                         out=torch.zeros_like(q))
        torch.cuda.synchronize()
        assert bool(out.isfinite().all())


@ROOM
def test_varlen_sequences_without_any_key(room):
    print(f"[attend] sequences without keys room {room}", flush=True)
    q = torch.randn(40, 8, 64, generator=torch.Generator().manual_seed(1)).to(BF)
    cache, _ = su.pool([1], [16], 2, 64, BF, 16, stale=NAN)
    cache.fill_(NAN)
    put = dict(dtype=torch.int32, device="cuda")
    rows, none = torch.tensor([0, 3, 3, 38], **put), torch.zeros(3, **put)
    for indices, indptr in ((torch.zeros(3 * (1 + room), **put), torch.arange(4, **put) * (1 + room)),
                            (torch.zeros(0, **put), torch.zeros(4, **put)), (torch.zeros(3, 2, **put), None)):
        out, lse = tsf.tree_sparse_attention_fwd_paged_varlen(
            q.cuda(), cache.cuda(), indices, q_indptr=rows, kv_lens=none, kv_indptr=indptr,
            out=torch.full((40, 8, 64), 3.0, dtype=BF, device="cuda"), return_lse=True)
        torch.cuda.synchronize()
        assert bool((out[:38] == 0).all()) and bool((lse[:38] == -torch.inf).all()) and bool((out[38:] == 3).all())


def test_varlen_fewer_keys_than_queries():
    print("[attend] fewer keys than query tokens", flush=True)
    # the first keys are the first tokens': columns past kv_len do not exist
    g = torch.Generator().manual_seed(3)
    cache, lists = su.pool([10], [6], 2, 64, BF, 16, stale=NAN)
    q = torch.randn(10, 4, 64, generator=g).to(BF)
    tree = su.tree_masks([10])
    ref, _, size, most = so.varlen_attention(q, cache, lists, tree, [10], [6])
    indices, indptr = su.tables(lists)
    q_indptr, kl = su.lengths([10], [6])
    got = tsf.tree_sparse_attention_fwd_paged_varlen(*_dev(q, cache, indices, tree), q_indptr=q_indptr.cuda(),
                                                     kv_lens=kl.cuda(), kv_indptr=indptr.cuda())
    assert bool(((got.double().cpu() - ref).abs() <= so.attention_tolerance(ref, size, most, BF, 6)).all())


def test_varlen_graph_follows_the_lengths():
    print("[attend] graph replays with other lengths", flush=True)
    q_lens, kv_lens = [12, 1, 30], [200, 33, 30]
    s = _attend(q_lens, kv_lens, page=64)
    kw = dict(q_indptr=s["q_indptr"], kv_lens=s["kv_lens"], kv_indptr=s["indptr"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(side):
        for _ in range(2):  # two graphs, a workspace of its own each
            tsf.tree_sparse_attention_fwd_paged_varlen(s["q"], s["cache"], s["indices"], s["tree"], **kw)
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                outs.append(tsf.tree_sparse_attention_fwd_paged_varlen(s["q"], s["cache"], s["indices"], s["tree"],
                                                                       **kw))
            graphs.append(g)
    torch.cuda.synchronize()
    for lens, rows in (([200, 33, 30], [0, 12, 13, 43]), ([150, 1, 29], [0, 5, 6, 30]), ([64, 0, 64], [0, 12, 12, 43])):
        s["kv_lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        s["q_indptr"].copy_(torch.tensor(rows, dtype=torch.int32))
        eager = tsf.tree_sparse_attention_fwd_paged_varlen(s["q"], s["cache"], s["indices"], s["tree"], **kw)
        for g, out in zip(graphs, outs):
            out.fill_(NAN)
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert _same(out[:rows[-1]], eager[:rows[-1]])


def test_varlen_shared_and_repeated_pages():
    print("[attend] pages shared by sequences, and twice in one list", flush=True)

    def edit(q, cache, lists, tree):
        lists[1][:4] = lists[0][:4]  # a common prefix
        lists[2][3] = lists[2][1]

    _attend([9, 20, 3], [105, 90, 80], edit=edit, stale=None)


def test_varlen_and_append_in_a_pool_past_32_bit_offsets():
    print("[attend] a pool of more than 2^31 elements", flush=True)
    q_lens, kv_lens, hkv, d = [17, 1], [200, 33], 8, 128
    g = torch.Generator().manual_seed(2)
    small, lists = su.pool(q_lens, kv_lens, hkv, d, BF, 16)
    n, total = small.shape[0], (1 << 31) // (2 * 16 * hkv * d) + 100
    big = torch.empty((total, 2, 16, hkv, d), dtype=BF, device="cuda")
    assert big.numel() > 1 << 31
    big[total - n:] = small.cuda()
    qkv = torch.randn(18, 32 + 2 * hkv, d, generator=g).to(BF).cuda()
    freq, positions = su.inv_freq(d).cuda(), torch.arange(18).cuda()
    outs = []
    for cache, shift in ((small.cuda(), 0), (big, total - n)):
        indices, indptr = su.tables([[p + shift for p in x] for x in lists])
        q_indptr, kl = su.lengths(q_lens, kv_lens)
        kw = dict(q_indptr=q_indptr.cuda(), kv_lens=kl.cuda(), kv_indptr=indptr.cuda())
        q = tsf.append_paged_kv(qkv[:, :32], qkv[:, 32:32 + hkv], qkv[:, 32 + hkv:], cache, indices.cuda(), positions,
                                freq, **kw)
        o = tsf.tree_sparse_attention_fwd_paged_varlen(q, cache, indices.cuda(), su.tree_masks(q_lens).cuda(), **kw)
        outs.append((q, o, cache[-n:]))
    torch.cuda.synchronize()
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_varlen_two_streams_at_once():
    print("[attend] two streams", flush=True)
    a = _attend([33, 9], [433, 109])
    b = _attend([2, 60], [900, 61], seed=5)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    torch.cuda.synchronize()
    for _ in range(4):
        for i, s in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i].append(tsf.tree_sparse_attention_fwd_paged_varlen(
                    s["q"], s["cache"], s["indices"], s["tree"], q_indptr=s["q_indptr"], kv_lens=s["kv_lens"],
                    kv_indptr=s["indptr"]))
    torch.cuda.synchronize()
    for i, s in enumerate((a, b)):
        for out in got[i]:
            assert torch.equal(out, s["out"])


# --------------------------------------------------------------------- append
APPEND = [
    # q lengths, kv lengths, keywords
    ([1], [1], dict()),
    ([3, 0, 5], [3, 0, 21], dict(interleaved=True)),                     # a page that ends inside the run
    ([40, 1], [56, 300], dict(dtype=FP, layout="HND", page=64, rot=64)),  # half of the head
    ([7, 9], [100, 33], dict(hq=14, hkv=2, d=64, dense=True, scaling=1.25)),
    ([20], [20], dict(rot=0)),                                           # no rotation at all
    ([5, 6], [37, 64], dict(hq=2, hkv=1, d=96, rot=32, pos32=True)),
    ([4], [4], dict(hq=2, hkv=1, d=256, rot=256, far=1000000)),          # far positions
    ([300, 1, 200], [310, 77, 200], dict(hq=4, hkv=1, d=64, far=131071)),
]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("case", APPEND, ids=[f"p{i}" for i in range(len(APPEND))])
def test_append(case, in_place):
    q_lens, kv_lens, kw = case
    print(f"[append] {case} in place {in_place}", flush=True)
    hq, hkv, d, dtype = kw.get("hq", 8), kw.get("hkv", 2), kw.get("d", 128), kw.get("dtype", BF)
    page, layout, rot = kw.get("page", 16), kw.get("layout", "NHD"), kw.get("rot", kw.get("d", 128))
    scaling, interleaved = kw.get("scaling", 1.0), kw.get("interleaved", False)
    n, pad = sum(q_lens), 3
    g = torch.Generator().manual_seed(n)
    cache, lists = su.pool(q_lens, kv_lens, hkv, d, dtype, page, layout, seed=n)
    qkv = torch.randn(n + pad, hq + 2 * hkv, d, generator=g).to(dtype)
    positions = torch.randint(0, 5000, (n + pad,), generator=g) + kw.get("far", 0)
    freq = su.inv_freq(rot)
    indices, indptr = su.tables(lists, kw.get("dense", False))
    q_indptr, kl = su.lengths(q_lens, kv_lens)
    ref = so.append(qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:], cache, lists, positions, freq, q_lens,
                    kv_lens, page, layout, interleaved, scaling)
    x, dc, di, dp, dqi, dkl, df, dpos = _dev(qkv, cache, indices, indptr, q_indptr, kl, freq, positions)
    if kw.get("pos32"):
        dpos = dpos.int()
    q = x[:, :hq]
    out = q if in_place else torch.full((n + pad, hq, d), 5.0, device="cuda", dtype=dtype)
    before = x.clone()
    got = tsf.append_paged_kv(q, x[:, hq:hq + hkv], x[:, hq + hkv:], dc, di, dpos, df, q_indptr=dqi, kv_lens=dkl,
                              kv_indptr=dp, kv_layout=layout, interleaved=interleaved, attention_scaling=scaling,
                              out=out)
    torch.cuda.synchronize()
    assert got is out
    qr, qs, new, size, written = ref
    # the angle is rounded to 2^-25 of a half turn and sine and cosine to a few units of 2^-24, two products and a
    # sum round in 32 bits: 2^-20 of the operands covers them; the result is rounded once
    u, e = torch.finfo(dtype).eps / 2, 2.0 ** -20
    assert bool(((got[:n].double().cpu() - qr[:n]).abs() <= u * (1 + e) * qr[:n].abs() + (e + u * e) * qs[:n]).all())
    if in_place:
        assert torch.equal(got[n:], before[n:, :hq]) and torch.equal(x[:, hq:], before[:, hq:])
    else:
        assert bool((got[n:] == 5.0).all()) and torch.equal(x, before)
    c = dc.cpu()
    assert torch.equal(c[~written], cache[~written])
    assert bool(((c.double() - new).abs() <= u * (1 + e) * new.abs() * (size > 0) + (e + u * e) * size).all())


def test_append_places_outside_the_lists_are_not_written():
    print("[append] places outside", flush=True)
    cache, lists = su.pool([6, 4], [20, 20], 2, 64, BF, 16)
    qkv = torch.randn(10, 8, 64, generator=torch.Generator().manual_seed(0)).to(BF)
    freq, positions = su.inv_freq(64), torch.arange(10)
    # sequence 0: keys 28 .. 33, its list ends at 32; sequence 1: 2 keys for 4 tokens, and pages outside the pool
    wild = [lists[0], [9999, -1]]
    q_lens, kv_lens = [6, 4], [34, 2]
    ref = so.append(qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], cache, wild, positions, freq, q_lens, kv_lens, 16)
    indices, indptr = su.tables(wild)
    q_indptr, kl = su.lengths(q_lens, kv_lens)
    x, dc, di, dp, dqi, dkl, df, dpos = _dev(qkv, cache, indices, indptr, q_indptr, kl, freq, positions)
    tsf.append_paged_kv(x[:, :4], x[:, 4:6], x[:, 6:], dc, di, dpos, df, q_indptr=dqi, kv_lens=dkl, kv_indptr=dp)
    torch.cuda.synchronize()
    written = ref[4]
    assert int(written.any(dim=(1, 3, 4)).sum()) == 4
    assert torch.equal(dc.cpu()[~written], cache[~written])
    assert float((dc.cpu().double() - ref[2])[written].abs().max()) < 0.05


# --------------------------------------------------------------------- select
def _logits(batch, beams, vocab, dtype, seed, peaks=4):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(batch, beams, vocab, generator=g) * 2.5
    at = torch.randint(vocab, (batch, beams, peaks), generator=g)
    x.scatter_add_(2, at, 8 * torch.rand(batch, beams, peaks, generator=g))
    scores = -torch.rand(batch, beams, generator=g) * 4
    return x.to(dtype), scores


def _select(logits, scores, k, states=()):
    got = tsf.beam_select(logits.cuda(), scores.cuda(), k, states=[s.cuda() for s in states])
    torch.cuda.synchronize()
    tokens, parents, best = so.beam_select(logits, scores, k)
    np.testing.assert_array_equal(got.tokens.cpu().numpy(), tokens)
    np.testing.assert_array_equal(got.parents.cpu().numpy(), parents)
    s = got.scores.double().cpu().numpy()
    live = np.isfinite(best)
    np.testing.assert_array_equal(np.isfinite(s), live)
    # one rounding of the 64-bit value
    assert (np.abs(s - best)[live] <= 2.0 ** -24 * np.abs(best[live]) + 1e-11).all()
    for state, new in zip(states, got.states):
        for b in range(logits.shape[0]):
            assert torch.equal(new[b].cpu(), state[b][torch.from_numpy(parents[b])])
    return got


@pytest.mark.parametrize("dtype", [BF, FP, torch.float32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("batch,beams,vocab,k", [(1, 1, 1, 1), (2, 1, 7, 7), (1, 1, 32000, 8), (3, 5, 1001, 10),
                                                 (2, 10, 9000, 64), (1, 64, 2049, 33), (5, 2, 8193, 1),
                                                 (130, 8, 515, 8), (1, 256, 40, 64), (52, 5, 20000, 10), (16, 8, 40001, 20),
                                                 (6, 10, 36000, 64), (3, 35, 4778, 31),
                                                 (1, 16, 160000, 64), (2, 11, 14164, 46)])
def test_select(dtype, batch, beams, vocab, k):
    print(f"[select] {dtype} {batch} {beams} {vocab} {k}", flush=True)
    logits, scores = _logits(batch, beams, vocab, dtype, seed=vocab + k)
    g = torch.Generator().manual_seed(1)
    states = (torch.randn(batch, beams, 24, generator=g).to(BF), torch.randint(9, (batch, beams, 3), generator=g),
              torch.rand(batch, beams, 5, 7, generator=g) > 0.5, torch.randn(batch, beams, generator=g))
    _select(logits, scores, k, states)


@pytest.mark.parametrize("dtype", [BF, torch.float32], ids=["bf16", "fp32"])
def test_select_ties_and_masked_vocabularies(dtype):
    print(f"[select] ties {dtype}", flush=True)
    inf = float("inf")
    logits, scores = _logits(8, 3, 9001, dtype, seed=4)
    logits[0] = 1.5                                  # every token alike: the lowest of the best beam
    logits[1] = logits[1].round()                    # many ties
    logits[2, :, 5:] = -inf                          # fewer tokens than k
    logits[2, 1] = -inf                              # a beam without any
    logits[3, 0, 17] = NAN
    logits[3, 2, ::2] = NAN
    logits[4, 1, [3, 8000]] = inf                    # tokens that take the whole mass
    logits[5] = -0.0
    logits[5, :, ::3] = 0.0
    logits[6] = torch.arange(9001).to(dtype)         # rising: the worst order to meet
    logits[7] = -inf                                 # nothing at all
    scores[0, 1] = scores[0, 2] = scores[0, 0]
    scores[3, 1] = NAN
    scores[4, 0] = inf
    scores[5, 0] = -inf
    _select(logits, scores, 20)
    _select(logits[:, :1].contiguous(), scores[:, :1].contiguous(), 64)


def test_select_more_ties_than_a_round_holds():
    print("[select] ties across beams", flush=True)
    logits = torch.full((2, 64, 2100), 0.25, dtype=BF)
    scores = torch.full((2, 64), -1.0)
    logits[1, 5:, 7] = 3.0  # and ties at the top
    _select(logits, scores, 64)
    for batch, beams, vocab in ((2, 256, 2100), (2, 64, 33000), (4, 15, 36000)):  # rows for tiles of each length
        logits = torch.full((batch, beams, vocab), -0.5, dtype=FP)
        scores = torch.zeros(batch, beams)
        scores[1, 7] = 0.25
        for k in (1, 3):
            _select(logits, scores, k)


def test_select_logits_past_32_bit_offsets():
    print("[select] logits of more than 2^31 elements apart", flush=True)
    logits, scores = _logits(2, 3, 5000, BF, seed=8)
    want = _select(logits, scores, 12)
    memory = torch.empty(((1 << 31) + 40000,), dtype=BF, device="cuda")
    far = memory.as_strided((2, 3, 5000), ((1 << 31) + 64, 5001, 1))
    far.copy_(logits)
    got = tsf.beam_select(far, scores.cuda(), 12)
    for a, b in zip(got[:3], want[:3]):
        assert torch.equal(a, b)


def test_select_states_moved_by_a_launch_of_their_own():
    print("[select] large states", flush=True)
    logits, scores = _logits(3, 4, 300, FP, seed=5)
    g = torch.Generator().manual_seed(3)
    _select(logits, scores, 9, (torch.randn(3, 4, 40001, generator=g), torch.randint(9, (3, 4, 7), generator=g)))


def test_select_strides_and_empty_batches():
    print("[select] strides", flush=True)
    logits, scores = _logits(3, 4, 777, FP, seed=9)
    want = _select(logits, scores, 6)
    wide = torch.full((3, 5, 1000), 50.0, dtype=FP)
    wide[:, 1:, 3:780] = logits
    got = tsf.beam_select(wide.cuda()[:, 1:, 3:780], scores.cuda(), 6)
    flipped = tsf.beam_select(logits.transpose(1, 2).contiguous().cuda().transpose(1, 2),
                              scores.t().contiguous().cuda().t(), 6)
    for x in (got, flipped):
        assert torch.equal(x.tokens, want.tokens) and torch.equal(x.parents, want.parents)
        assert torch.equal(x.scores, want.scores)
    none = tsf.beam_select(logits.cuda()[:0], scores.cuda()[:0], 6, states=(torch.zeros(0, 4, 8).cuda(),))
    assert none.tokens.shape == (0, 6) and none.states[0].shape == (0, 6, 8)


def test_select_in_a_graph():
    print("[select] graph", flush=True)
    logits, scores = _logits(2, 4, 30001, BF, seed=2)
    state = torch.randn(2, 4, 64)
    x, c, h = logits.cuda(), scores.cuda(), state.cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        tsf.beam_select(x, c, 5, states=(h,))
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            got = tsf.beam_select(x, c, 5, states=(h,))
    torch.cuda.synchronize()
    for rep in range(3):
        x.copy_(torch.roll(logits, rep, 2).cuda())
        eager = tsf.beam_select(x, c, 5, states=(h,))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip((*got[:3], got.states[0]), (*eager[:3], eager.states[0])):
            assert torch.equal(a, b)


# ---------------------------------------------------------------- the chain
def test_draft_append_attend():
    """Two steps of a draft: beams selected from logits, their tokens appended as a tree behind prefixes of
    different lengths, attended to; every stage against the plain forms fed with the kernels' inputs."""
    print("[chain] draft, append, attend", flush=True)
    batch, beams, vocab, hq, hkv, d, page = 3, 4, 5003, 8, 2, 128, 16
    g = torch.Generator().manual_seed(0)
    prefix = [33, 7, 260]
    levels = 3
    q_lens = [1 + beams * levels] * batch  # the root and three levels of beams
    kv_lens = [p + m for p, m in zip(prefix, q_lens)]
    cache, lists = su.pool(q_lens, kv_lens, hkv, d, BF, page)
    freq = su.inv_freq(d)
    scores = torch.zeros(batch, 1)
    rows = torch.ones(batch, 1, 1, dtype=torch.bool)  # tree rows of the current beams: their ancestors
    mask = torch.zeros(batch, q_lens[0], q_lens[0], dtype=torch.bool)
    mask[:, 0, 0] = True
    depth = torch.zeros(batch, q_lens[0], dtype=torch.int64)
    for level in range(levels):
        width = 1 if level == 0 else beams
        logits = (torch.randn(batch, width, vocab, generator=g) * 3).to(BF)
        best = _select(logits, scores, beams, states=(rows,))
        scores = best.scores.cpu()
        rows = torch.cat((best.states[0].cpu(), torch.eye(beams, dtype=torch.bool).expand(batch, -1, -1)), dim=2)
        first = 1 + level * beams
        mask[:, first:first + beams, :first + beams] = rows
        depth[:, first:first + beams] = level + 1
    positions = (torch.tensor(prefix)[:, None] + depth).reshape(-1)
    n = sum(q_lens)
    qkv = torch.randn(n, hq + 2 * hkv, d, generator=g).to(BF)
    indices, indptr = su.tables(lists)
    q_indptr, kl = su.lengths(q_lens, kv_lens)
    x, dc, di, dp, dqi, dkl, df, dpos, dm = _dev(qkv, cache, indices, indptr, q_indptr, kl, freq, positions, mask)
    lists_kw = dict(q_indptr=dqi, kv_lens=dkl, kv_indptr=dp)
    q = tsf.append_paged_kv(x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], dc, di, dpos, df, **lists_kw)
    o = tsf.tree_sparse_attention_fwd_paged_varlen(q, dc, di, dm, **lists_kw)
    torch.cuda.synchronize()
    qr, qs, new, size, _ = so.append(qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:], cache, lists, positions,
                                     freq, q_lens, kv_lens, page)
    u = torch.finfo(BF).eps / 2
    assert bool(((q.double().cpu() - qr).abs() <= 1.01 * u * qr.abs() + 2.0 ** -19 * qs).all())
    assert bool(((dc.double().cpu() - new).abs() <= 1.01 * u * new.abs() + 2.0 ** -19 * size).all())
    ref, _, vsize, most = so.varlen_attention(q.cpu(), dc.cpu(), lists, mask, q_lens, kv_lens)
    assert bool(((o.double().cpu() - ref).abs() <= so.attention_tolerance(ref, vsize, most, BF, max(kv_lens))).all())
