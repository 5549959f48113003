"""The operators of a drafted decoding step on the GPU against their definitions in 64 bits."""
import math
import random

import numpy as np
import pytest
import torch

from oracle import draft_oracle as orc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16


@pytest.fixture(scope="module")
def be():
    from rivoli_b200 import backend
    backend.lib()
    return backend


def i32(v, device=DEV):
    return torch.tensor(v, dtype=torch.int32, device=device)


def u64(t):
    return [m + (1 << 64) if m < 0 else m for m in t.tolist()]


# --- rotary positions ------------------------------------------------------------------------------------------------
def rope_tolerance(x, want, scale):
    """Half a bf16 step of the result, and 2^-21 of the pair's size for the 32-bit cosines, sines and products: the angle's last bit
    at pi (2^-23 and its rounding to 32 bits), a few steps of the functions, three roundings of the sum."""
    half = x.shape[-1] // 2
    size = np.abs(x).max(-1, keepdims=True) * scale * np.ones(2 * half)
    return 2.0 ** -8 * np.abs(want) + 2.0 ** -20 * size


@pytest.mark.parametrize("layout", ["adjacent", "half", "split"])
@pytest.mark.parametrize("seg, width, off, heads, rows", [
    (64, 256, 192, 64, 3), (64, 64, 0, 1, 1), (128, 128, 0, 5, 700), (16, 48, 16, 7, 2), (48, 56, 8, 3, 5), (512, 512, 0, 2, 3),
    (20, 24, 4, 4, 9), (64, 67, 3, 3, 4), (2, 2, 0, 1, 1), (6, 8, 1, 300, 2), (96, 160, 64, 33, 40), (500, 502, 2, 2, 3)])
def test_rope_against_the_definition(be, layout, seg, width, off, heads, rows):
    g = torch.Generator().manual_seed(seg * 1000 + width + rows)
    q, k = (torch.randn(s, generator=g, dtype=torch.float32).to(BF) for s in ((rows, heads, width), (rows, width)))
    pos = torch.randint(-5, 1 << 20, (rows,), generator=g, dtype=torch.int32)
    pos[0] = (1 << 31) - 1 if rows > 1 else 7
    f, scale = be.rope_frequencies(seg, 10000.0, "yarn" if seg == 64 else "none", 4.0 if seg == 64 else 1.0)
    want_q = orc.rope(q.double().numpy()[..., off:off + seg], pos.numpy(), f, layout, scale)
    want_k = orc.rope(k.double().numpy()[:, None, off:off + seg], pos.numpy(), f, layout, scale)
    tol_q = rope_tolerance(q.double().numpy()[..., off:off + seg], want_q, scale)
    tol_k = rope_tolerance(k.double().numpy()[:, None, off:off + seg], want_k, scale)
    inv = torch.from_numpy(f).to(DEV)
    # out of place, and in place in the middle of wider rows
    dq, dk = q.to(DEV), k.to(DEV)
    oq, ok = torch.zeros((rows, heads, seg), dtype=BF, device=DEV), torch.zeros((rows, seg), dtype=BF, device=DEV)
    sq, sk = dq[..., off:off + seg], dk[..., off:off + seg]
    be.launch_rope_rows_bf16(be.rope_vecs(sq, oq), be.rope_vecs(sk, ok), rows, pos.to(DEV), inv, seg, be.ROPE_LAYOUTS[layout], scale)
    assert torch.equal(dq.cpu(), q) and torch.equal(dk.cpu(), k)
    assert (np.abs(oq.double().cpu().numpy() - want_q) <= tol_q).all()
    assert (np.abs(ok.double().cpu().numpy()[:, None] - want_k) <= tol_k).all()
    be.launch_rope_rows_bf16(be.rope_vecs(sq), None, rows, pos.to(DEV), inv, seg, be.ROPE_LAYOUTS[layout], scale)
    be.launch_rope_rows_bf16(be.rope_vecs(sk), None, rows, pos.to(DEV), inv, seg, be.ROPE_LAYOUTS[layout], scale)
    assert torch.equal(sq.cpu(), oq.cpu()) and torch.equal(sk.cpu(), ok.cpu())
    dq[..., off:off + seg], dk[..., off:off + seg] = q[..., off:off + seg].to(DEV), k[..., off:off + seg].to(DEV)
    assert torch.equal(dq.cpu(), q) and torch.equal(dk.cpu(), k)      # nothing beside the segments was written


def test_rope_split_is_the_single_vector_operator(be):
    """The same permutation and angles as ``rope_interleave`` on f32 vectors, to bf16's last bit."""
    x = torch.randn((5, 64), generator=torch.Generator().manual_seed(3)).to(BF)
    f, _ = be.rope_frequencies(64)
    y = x.to(DEV)[:, None].clone()
    be.launch_rope_rows_bf16(be.rope_vecs(y), None, 5, i32([123] * 5), torch.from_numpy(f).to(DEV), 64, be.ROPE_LAYOUTS["split"])
    z = x.float().to(DEV)
    be.launch_rope_interleave(z, 5, 64, 64, 123, 10000.0)
    assert (y[:, 0].float() - z).abs().le(2.0 ** -8 * z.abs() + 2.0 ** -18).all()


def test_rope_negative_and_zero_strides(be):
    """Rows read backwards, and one vector read for several."""
    x = torch.randn((4, 64), generator=torch.Generator().manual_seed(4)).to(BF).to(DEV)
    f = torch.from_numpy(be.rope_frequencies(64)[0]).to(DEV)
    out = torch.zeros((4, 3, 64), dtype=BF, device=DEV)
    be.launch_rope_rows_bf16((x.data_ptr() + 3 * 128, out, -64, 0, 192, 64, 3), None, 4, i32([9, 8, 7, 6]), f, 64, 1)
    one = torch.zeros((4, 64), dtype=BF, device=DEV)
    be.launch_rope_rows_bf16(be.rope_vecs(x, one), None, 4, i32([6, 7, 8, 9]), f, 64, 1)
    assert all(torch.equal(out[:, h], one.flip(0)) for h in range(3))


# --- tree attention ----------------------------------------------------------------------------------------------------
class Cache:
    """Pools of random rows and a shuffled block table for sequences of the given lengths (prefix + nodes)."""

    def __init__(self, seed, lens, page, kvl=512, rope=64, spread=1.0):
        g = np.random.RandomState(seed)
        self.page, self.W = page, kvl + rope
        need = [max(1, -(-n // page)) for n in lens]
        self.n_pages = sum(need) + 3
        rows = self.n_pages * page
        x = g.randn(rows, self.W) * np.exp(spread * g.randn(rows, 1))
        scale = (np.abs(x).max(1) / 448).astype(np.float32)
        self.codes = torch.from_numpy((x / scale[:, None]).astype(np.float32)).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
        self.scale = scale
        order = g.permutation(self.n_pages).astype(np.int32)
        self.table = np.full((len(lens), max(need)), -1, dtype=np.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n

    def dev(self):
        return [torch.from_numpy(a).to(DEV) for a in (self.codes, self.scale, self.table)]


def masks_of(host, T, kind):
    if kind == "chain":
        return [(1 << (j + 1)) - 1 for j in range(T)]
    if kind == "empty":
        return [0] * T
    if kind == "all":
        return [(1 << 64) - 1] * T
    if kind == "any":
        return [host.getrandbits(64) if host.random() < 0.8 else 0 for _ in range(T)]
    parents = [-1] + [host.randrange(max(0, j - 4), j) for j in range(1, T)]
    bits = []
    for j, p in enumerate(parents):
        bits.append((bits[p] if p >= 0 else 0) | 1 << j)
    return bits


def signed(masks):
    return torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks], dtype=torch.int64, device=DEV)


def run_tree(be, cache, H, prefix, trees, masks, rows=None, n_rows=None, tree_pos=None, kvl=512, rope=64, q_scale=1.0, scratch=True,
             seed=0, stream=None, softmax_scale=None):
    """Launches one call, compares it with the definition, returns (out, lse, arguments, tolerances by sequence)."""
    start = np.concatenate(([0], np.cumsum(trees))).tolist()
    N, B = start[-1], len(trees)
    g = be.DsaGeom.make(n_heads=H, kv_lora=kvl, rope_dim=rope, page_tokens=cache.page, max_pages_per_seq=cache.table.shape[1],
                        n_pool_pages=cache.n_pages, softmax_scale=softmax_scale)
    q = (torch.randn((N, H, cache.W), generator=torch.Generator().manual_seed(seed)) * q_scale).to(BF)
    codes, scale, table = cache.dev()
    tree_pos = prefix if tree_pos is None else tree_pos
    out = torch.full((N + 1, H, kvl), 7.0, dtype=BF, device=DEV)
    lse = torch.full((N + 1, H), 7.0, device=DEV)
    sc = scratch if torch.is_tensor(scratch) else torch.zeros(be.mla_tree_attend_scratch_bytes(g, B, N), dtype=torch.uint8, device=DEV) if scratch else None
    r = None if rows is None else i32([[v - (1 << 32) if v >> 31 else v for v in row] for row in rows])
    counts = None if n_rows is None else i32(n_rows)
    args = [g, q.to(DEV), codes, scale, table, r, 0 if r is None else r.shape[1], counts, i32(tree_pos), i32(start), signed(masks), B, N, out, lse, sc, stream]
    torch.cuda.synchronize()
    be.launch_mla_tree_attend_paged_bf16(*args)
    torch.cuda.synchronize()
    if sc is not None:
        be.mla_tree_attend_status(g, sc)
    assert (out[N] == 7).all() and (lse[N] == 7).all()
    got, got_lse = out[:N].double().cpu().numpy(), lse[:N].double().cpu().numpy()
    cap = cache.table.shape[1] * cache.page
    err2 = norm2 = 0.0
    tols = []
    for b in range(B):
        T, a = trees[b], start[b]
        if not T:
            continue
        dense = rows is None or rows[b][0] == 0xffffffff
        n = (prefix[b] if n_rows is None else n_rows[b])
        n = max(0, min(n, cap if dense else len(rows[b])))
        at = orc.tree_rows(cache.table[b], cache.page, cache.n_pages, n, None if dense else rows[b], tree_pos[b], T)
        unit = 2.0 ** -8 / math.sqrt(3)
        want, want_lse, by_score, lse_by, by_weight, weight, step, by_step = orc.tree_attend(
            q[a:a + T].double().numpy(), cache.codes, cache.scale, at, n, masks[a:a + T], float(np.float32(g.softmax_scale)), kvl, unit)
        # The query as two 8-bit terms is off by up to 2^-8 relative in every entry (uniform: deviation 2^-8 / sqrt 3), which moves the
        # scores, six deviations at most; the weights as two terms by up to 2^-8 each; the result by half a bf16 step, 2^-8.
        # 2^-16: 32-bit exponents and sums. A weight times its row's scale is at most 2^8 and the largest at least 2^5 in units whose
        # 8-bit terms go down in steps of 2^-9: all are off by up to 2^-10 besides, 2^-15 of the largest.
        tol = 2.0 ** -8 * np.abs(want) + (2.0 ** -8 + 2.0 ** -16) * weight + 6 * by_score + 2.0 ** -15 * step + 1e-30
        assert (np.abs(got[a:a + T] - want) <= tol).all(), (b, (np.abs(got[a:a + T] - want) / tol).max())
        none = np.isinf(want_lse)
        assert (got_lse[a:a + T][none] == -np.inf).all() and (got[a:a + T][none] == 0).all()
        lse_tol = 6 * lse_by + 2.0 ** -16 + 2.0 ** -20 * np.abs(np.where(none, 0, want_lse))
        assert (np.abs(got_lse[a:a + T][~none] - want_lse[~none]) <= lse_tol[~none]).all()
        tols.append((tol, lse_tol))
        err2 += ((got[a:a + T] - want) ** 2).sum()
        norm2 += ((unit * want) ** 2 + by_score ** 2 + by_weight ** 2 + (2.0 ** -15 * by_step) ** 2).sum()
    # the squares add up; a sum over few heads and rows may come out at three times its mean's root
    assert math.sqrt(err2) <= 3 * math.sqrt(norm2) + 1e-30
    return out, lse, args, tols


@pytest.mark.parametrize("H", [64, 16])
@pytest.mark.parametrize("T, n, kind", [
    (1, 0, "chain"), (1, 1, "chain"), (1, 63, "tree"), (2, 64, "chain"), (3, 61, "tree"), (5, 257, "tree"), (64, 0, "tree"), (64, 65, "tree"),
    (64, 64, "any"), (17, 100, "any"), (33, 0, "any"), (7, 0, "empty"), (7, 130, "empty"), (9, 55, "all"), (31, 1000, "tree"), (64, 127, "chain")])
def test_tree_of_one_sequence(be, H, T, n, kind):
    host = random.Random(T * 1000 + n)
    run_tree(be, Cache(T + n, [n + T], 64), H, [n], [T], masks_of(host, T, kind), seed=T)


@pytest.mark.parametrize("H, page", [(64, 64), (64, 16), (48, 32), (1, 128), (128, 64), (3, 8), (40, 1)])
def test_ragged_trees(be, H, page):
    """Sequences without nodes, without a prefix, and of every size between; a table wider than most rows need."""
    host = random.Random(H * page)
    trees = [3, 0, 64, 1, 17, 0, 8, 33, 2]
    prefix = [200, 50, 0, 1, 63, 64, 700, 129, 65]
    masks = [m for t in trees for m in masks_of(host, t, host.choice(("tree", "any")))]
    run_tree(be, Cache(H + page, [p + t for p, t in zip(prefix, trees)], page), H, prefix, trees, masks, seed=H)


def test_tree_over_a_selection(be):
    """Listed rows, a row listed twice, the dense marker, counts past the list's end and below zero, tokens off the table."""
    host = random.Random(5)
    trees, prefix = [4, 8, 3, 5, 2, 6], [900, 500, 300, 400, 100, 64]
    k = 200
    rows = [sorted(host.sample(range(p), min(p, k))) for p in prefix]
    rows = [r + [1 << 30] * (k - len(r)) for r in rows]
    rows[1][0] = 0xffffffff
    rows[2][5] = rows[2][6]
    rows[3][7] = 0xfffffff0
    rows[4][3] = 100000
    n_rows = [200, 450, 200, 1000, 100, -3]
    masks = [m for t in trees for m in masks_of(host, t, "tree")]
    run_tree(be, Cache(9, [p + t for p, t in zip(prefix, trees)], 64), 64, prefix, trees, masks, rows=rows, n_rows=n_rows)


def test_dense_prefix_shorter_than_the_position(be):
    host = random.Random(6)
    run_tree(be, Cache(10, [300, 300], 32), 64, [280, 270], [9, 30], masks_of(host, 9, "tree") + masks_of(host, 30, "tree"), n_rows=[100, 0])


def test_unmapped_pages_are_seen_by_nobody(be):
    host = random.Random(7)
    cache = Cache(11, [500, 400, 90], 64)
    cache.table[0, 2] = -1
    cache.table[0, 5] = cache.n_pages
    cache.table[1, 6] = -7                       # the page that most of the tree lies on
    cache.table[2, :] = -1                       # nothing at all
    masks = [m for t in (6, 10, 5) for m in masks_of(host, t, "tree")]
    run_tree(be, cache, 64, [490, 383, 80], [6, 10, 5], masks)


@pytest.mark.parametrize("kvl", [512, 256])
def test_a_node_that_is_nan_reaches_its_descendants_alone(be, kvl):
    """NaN codes, and a NaN scale, in rows of the tree: nodes that do not see them give what they gave."""
    cache = Cache(21, [100, 70], 64, kvl)
    masks = [0b1, 0b11, 0b101, 0b1101, 0b10011] + [0b1, 0b11, 0b101]
    out, lse, args, _ = run_tree(be, cache, 64, [95, 62], [5, 3], masks, kvl=kvl)
    at = orc.tree_rows(cache.table[0], 64, cache.n_pages, 0, None, 95, 5)
    bt = orc.tree_rows(cache.table[1], 64, cache.n_pages, 0, None, 62, 3)
    codes, scale = args[2].clone(), args[3].clone()
    codes[at[1], 7], codes[at[1], 300], codes[at[3], kvl + 5] = 0x7f, 0xff, 0x7f       # seen by nodes 1 and 4, and by node 3
    scale[bt[1]], scale[bt[2]] = math.nan, math.inf                                    # by nodes 1 and 2 of the second
    again, lse2 = torch.zeros_like(out), torch.zeros_like(lse)
    be.launch_mla_tree_attend_paged_bf16(args[0], args[1], codes, scale, *args[4:13], again, lse2, *args[15:])
    for node in (0, 2, 5):
        assert torch.equal(again[node], out[node]) and torch.equal(lse2[node], lse[node])
    for node in (1, 3, 4, 6, 7):
        assert lse2[node].isnan().all() or (lse2[node] == math.inf).all() or again[node].isnan().any(), node


@pytest.mark.parametrize("kvl", [512, 256])
@pytest.mark.parametrize("where", ["code", "scale", "query"])
def test_a_node_that_sees_nan_alone(be, kvl, where):
    """Nothing but NaN is not nothing: the node's output and log-sum-exp are NaN, and the next sequence's are what they are."""
    cache = Cache(22, [1, 9], 64, kvl)
    out, lse, args, _ = run_tree(be, cache, 8, [0, 8], [1, 1], [1, 1], kvl=kvl)
    at = orc.tree_rows(cache.table[0], 64, cache.n_pages, 0, None, 0, 1)
    q, codes, scale = args[1].clone(), args[2].clone(), args[3].clone()
    if where == "code":
        codes[at[0]] = 0x7f
    elif where == "scale":
        scale[at[0]] = math.nan
    else:
        q[0] = math.nan
    again, lse2 = torch.zeros_like(out), torch.zeros_like(lse)
    be.launch_mla_tree_attend_paged_bf16(args[0], q, codes, scale, *args[4:13], again, lse2, *args[15:])
    assert again[0].isnan().all() and lse2[0].isnan().all()
    assert torch.equal(again[1], out[1]) and torch.equal(lse2[1], lse[1])


def test_rows_that_no_node_may_see_do_not_matter(be):
    """NaN codes and infinite scales in rows that only masks hide, and behind the last one."""
    cache = Cache(12, [200, 64], 64)
    host = random.Random(8)
    masks = [0b1, 0b10, 0b101] + masks_of(host, 2, "chain")
    out, lse, args, _ = run_tree(be, cache, 64, [150, 60], [3, 2], masks)
    page, slot = cache.table[0, (150 + 3) // 64], (150 + 3) % 64
    codes, scale = args[2].clone(), args[3].clone()
    codes[page * 64 + slot:(page + 1) * 64] = 0x7f
    scale[page * 64 + slot:(page + 1) * 64] = math.inf
    again, lse2 = torch.zeros_like(out), torch.zeros_like(lse)
    be.launch_mla_tree_attend_paged_bf16(args[0], args[1], codes, scale, *args[4:13], again, lse2, *args[15:])
    assert torch.equal(again[:5], out[:5]) and torch.equal(lse2[:5], lse[:5])


@pytest.mark.parametrize("kvl, rope, H", [(512, 128, 5), (256, 64, 16), (128, 16, 64), (384, 32, 7), (512, 48, 33)])
def test_other_geometries(be, kvl, rope, H):
    host = random.Random(kvl + rope)
    trees, prefix = [5, 1, 20], [70, 0, 33]
    masks = [m for t in trees for m in masks_of(host, t, "tree")]
    run_tree(be, Cache(13, [p + t for p, t in zip(prefix, trees)], 16, kvl, rope), H, prefix, trees, masks, kvl=kvl, rope=rope)


def test_without_scratch(be):
    host = random.Random(14)
    run_tree(be, Cache(14, [140], 64), 64, [130], [9], masks_of(host, 9, "tree"), scratch=False)


@pytest.mark.parametrize("q_scale", [0.0, 1e-6, 30.0])
def test_flat_and_peaked_scores(be, q_scale):
    """Peaked: one row takes it all, and references move by many binades from tile to tile."""
    host = random.Random(15)
    run_tree(be, Cache(15, [700], 64, spread=0.3), 64, [690], [4], masks_of(host, 4, "tree"), q_scale=q_scale)


@pytest.mark.parametrize("H, q_scale, spread", [(64, 1.0, 1.0), (16, 1.0, 0.3), (64, 7.3, 0.3), (64, 1e-30, 1.0)])
def test_scores_keep_the_querys_bits(be, H, q_scale, spread):
    """A bf16 is two e4m3 terms in full if it is within 2^-10 of its row's largest, and off by at most 2^-18 of that if not: the sums of
    the softmax, which nothing else rounds to fewer than 32 bits, show it. Sums in the tensor cores: 18 steps of 32 products for each
    of two terms and their own sum, each rounded or cut to 24 bits, 2^-23; 2^-18 for the exponentials and the sum over 1,106 rows."""
    cache = Cache(21, [1106], 64, spread=spread)
    out, lse, args, _ = run_tree(be, cache, H, [1100], [6], masks_of(random.Random(21), 6, "chain"), q_scale=q_scale, seed=3)
    at = orc.tree_rows(cache.table[0], cache.page, cache.n_pages, 1100, None, 1100, 6)
    k = torch.from_numpy(cache.codes).view(torch.float8_e4m3fn).double().numpy()[at] * cache.scale[at].astype(np.float64)[:, None]
    q = args[1].double().cpu().numpy()
    scale = float(np.float32(args[0].softmax_scale))
    for t in range(6):
        seen = slice(0, 1100 + t + 1)
        s = q[t] @ k[seen].T * scale
        top = s.max(1, keepdims=True)
        want = top[:, 0] + np.log(np.exp(s - top).sum(1))
        off = (2.0 ** -18 * np.abs(q[t]).max(1, keepdims=True) * np.abs(k[seen]).sum(1) + 37 * 2.0 ** -23 * (np.abs(q[t]) @ np.abs(k[seen]).T)) * scale
        # what a row's score is off by moves the sum by its share of it
        tol = (np.exp(s - top) / np.exp(s - top).sum(1, keepdims=True) * off).sum(1) + 2.0 ** -18 + 2.0 ** -22 * np.abs(want)
        assert (np.abs(lse[t].double().cpu().numpy() - want) <= tol).all(), (np.abs(lse[t].double().cpu().numpy() - want) / tol).max()


@pytest.mark.parametrize("kvl, rope", [(512, 64), (256, 64)])
def test_scales_from_tiny_to_huge(be, kvl, rope):
    """Row scales of 2^-90 and 2^60 (the query the other way round there, so that scores stay small); below 2^-100 the outputs may vanish
    but nothing overflows; rows of scale zero are not there."""
    host = random.Random(24)
    masks = masks_of(host, 5, "tree")
    for e in (-90, 60):
        cache = Cache(24, [205], 64, kvl, rope, spread=0.3)
        cache.scale = np.ldexp(cache.scale, e).astype(np.float32)
        run_tree(be, cache, 24, [200], [5], masks, kvl=kvl, rope=rope, q_scale=2.0 ** min(0, -e))
    cache = Cache(25, [205], 64, kvl, rope, spread=0.3)
    keep = cache.scale.copy()
    cache.scale = np.ldexp(keep, -118).astype(np.float32)
    at = orc.tree_rows(cache.table[0], 64, cache.n_pages, 200, None, 200, 5)
    cache.scale[at[:50]] = 0.0
    g = be.DsaGeom.make(n_heads=24, kv_lora=kvl, rope_dim=rope, max_pages_per_seq=4, n_pool_pages=cache.n_pages)
    q = torch.randn((5, 24, kvl + rope), generator=torch.Generator().manual_seed(1)).to(BF).to(DEV)
    out, lse = torch.zeros((5, 24, kvl), dtype=BF, device=DEV), torch.zeros((5, 24), device=DEV)
    sc = torch.zeros(be.mla_tree_attend_scratch_bytes(g, 1, 5), dtype=torch.uint8, device=DEV)
    be.launch_mla_tree_attend_paged_bf16(g, q, *cache.dev(), None, 0, None, i32([200]), i32([0, 5]), signed(masks), 1, 5, out, lse, sc)
    torch.cuda.synchronize()
    seen = torch.tensor([150 + bin(m).count("1") for m in masks], device=DEV, dtype=torch.float64)
    # scores below 2^-100: the log-sum-exp is the logarithm of the rows' number; 32 bits of an exponent of about 110 and of the sum
    assert ((lse.double() - seen.log()[:, None]).abs() <= 2.0 ** -15).all()
    assert (out.float().abs() <= float(cache.scale.max()) * 448).all()


def test_long_cache(be):
    """One sequence split over the whole chip, and short ones beside it."""
    host = random.Random(16)
    trees, prefix = [2, 5, 1], [20011, 40, 1500]
    masks = [m for t in trees for m in masks_of(host, t, "tree")]
    run_tree(be, Cache(16, [p + t for p, t in zip(prefix, trees)], 64), 64, prefix, trees, masks)


@pytest.mark.parametrize("page, listed", [(64, False), (16, False), (64, True)])
def test_rows_past_four_gigabytes(be, page, listed):
    """The same pages at the end of a pool of 4.4 GB and in a small one: the same bits, and the rows move there too."""
    host = random.Random(23)
    prefix, trees, H = [700, 90], [5, 9], 16
    cache = Cache(23, [p + t for p, t in zip(prefix, trees)], page)
    masks = [m for t in trees for m in masks_of(host, t, "tree")]
    rows = [sorted(host.sample(range(p), 80)) for p in prefix] if listed else None
    out, lse, args, _ = run_tree(be, cache, H, prefix, trees, masks, rows=rows, n_rows=[80, 80] if listed else None)
    g, codes, scale, table = args[0], args[2], args[3], args[4]
    big_pages = 7_700_000 // page
    shift = big_pages - cache.n_pages
    big = be.DsaGeom.make(n_heads=H, page_tokens=page, max_pages_per_seq=table.shape[1], n_pool_pages=big_pages)
    far = torch.empty((big_pages * page, cache.W), dtype=torch.uint8, device=DEV)
    far_scale = torch.empty(big_pages * page, device=DEV)
    far[shift * page:], far_scale[shift * page:] = codes, scale
    far_table = torch.where(table >= 0, table + shift, table)
    again, lse2 = torch.zeros_like(out), torch.zeros_like(lse)
    be.launch_mla_tree_attend_paged_bf16(big, args[1], far, far_scale, far_table, *args[5:13], again, lse2, args[15])
    torch.cuda.synchronize()
    be.mla_tree_attend_status(big, args[15])
    assert torch.equal(again[:14], out[:14]) and torch.equal(lse2[:14], lse[:14])
    path = torch.tensor([[0, 2, 4], [0, 5, 8]], dtype=torch.int32, device=DEV)
    for G, pool, sc, tab in ((g, codes, scale, table), (big, far, far_scale, far_table)):
        be.launch_kv_commit_paged(G, be.commit_layers([(pool, sc, None, None)]), 1, tab, args[8], path, 3, i32([3, 3]), 2, None, None)
    torch.cuda.synchronize()
    assert torch.equal(far[shift * page:], codes) and torch.equal(far_scale[shift * page:], scale)
    assert not torch.equal(codes.cpu(), torch.from_numpy(cache.codes))


def test_one_scratch_for_calls_of_every_shape(be):
    """What one call leaves in the scratch is nothing to the next: long after short, one block after many, and back."""
    host = random.Random(22)
    shared = torch.zeros(64 << 20, dtype=torch.uint8, device=DEV)
    g = be.DsaGeom.make(max_pages_per_seq=4, n_pool_pages=8)
    assert be.mla_tree_attend_scratch_bytes(g, 1, 1) <= shared.numel()
    for trees, prefix, H in (([2], [9000], 64), ([1] * 200, [70 + i for i in range(200)], 64), ([3, 1], [10, 300], 16), ([64] * 5, [600] * 5, 64),
                             ([1], [5], 64), ([33], [5000], 64), ([2] * 40, [1000 - 20 * i for i in range(40)], 64)):
        masks = [m for t in trees for m in masks_of(host, t, "tree")]
        run_tree(be, Cache(len(trees), [p + t for p, t in zip(prefix, trees)], 64), H, prefix, trees, masks, scratch=shared)


def test_many_sequences(be):
    host = random.Random(17)
    trees, prefix = [1 + i % 3 for i in range(300)], [i % 90 for i in range(300)]
    masks = [m for t in trees for m in masks_of(host, t, "tree")]
    run_tree(be, Cache(17, [p + t for p, t in zip(prefix, trees)], 16), 16, prefix, trees, masks)


def test_same_call_same_bits(be):
    host = random.Random(18)
    trees, prefix = [7, 12, 40], [3000, 5000, 100]
    masks = [m for t in trees for m in masks_of(host, t, "tree")]
    out, lse, args, _ = run_tree(be, Cache(18, [p + t for p, t in zip(prefix, trees)], 64), 64, prefix, trees, masks)
    for _ in range(3):
        again, lse2 = torch.zeros_like(out), torch.zeros_like(lse)
        be.launch_mla_tree_attend_paged_bf16(*args[:13], again, lse2, *args[15:])
        assert torch.equal(again[:59], out[:59]) and torch.equal(lse2[:59], lse[:59])


def test_one_node_is_the_decode_steps_attention(be):
    """A tree of one node is the attention of a decode step over prefix + 1 rows."""
    cache = Cache(19, [600, 200], 64)
    out, lse, args, tols = run_tree(be, cache, 64, [599, 199], [1, 1], [1, 1])
    g = args[0]
    want, want_lse = torch.zeros_like(out[:2]), torch.zeros_like(lse[:2])
    scratch = torch.zeros(256, dtype=torch.uint8, device=DEV)
    be.launch_attend_paged_bf16(g, args[1], args[2], args[3], args[4], None, 0, i32([600, 200]), 2, want, None, want_lse, scratch)
    for b, (tol, lse_tol) in enumerate(tols):                 # both kernels split q and the weights: each is within these
        assert (np.abs((out[b].double() - want[b].double()).cpu().numpy()) <= 2 * tol[0]).all()
        assert (np.abs((lse[b] - want_lse[b]).double().cpu().numpy()) <= 2 * lse_tol[0]).all()


def test_tree_captured_and_on_another_stream(be):
    host = random.Random(20)
    trees, prefix = [5, 30], [400, 2000]
    masks = [m for t in trees for m in masks_of(host, t, "tree")]
    side = torch.cuda.Stream()
    out, lse, args, _ = run_tree(be, Cache(20, [p + t for p, t in zip(prefix, trees)], 64), 64, prefix, trees, masks, stream=side)
    again, lse2 = torch.zeros_like(out), torch.zeros_like(lse)
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            be.launch_mla_tree_attend_paged_bf16(*args[:13], again, lse2, args[15], torch.cuda.current_stream())
    for _ in range(2):
        again.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(again[:35], out[:35]) and torch.equal(lse2[:35], lse[:35])


# --- verification -----------------------------------------------------------------------------------------------------
def run_verify(be, counts, parents, token, target, draft, u, u_next, most, vocab=None):
    start = np.concatenate(([0], np.cumsum(counts))).tolist()
    B, V = len(counts), vocab or target.shape[1]
    path = torch.full((B + 1, most), -9, dtype=torch.int32, device=DEV)
    n_path, nxt = i32([-9] * (B + 1)), i32([-9] * (B + 1))
    be.launch_draft_verify(i32(start), i32(parents or [0]), i32(token or [0]), target, target.stride(0), draft, 0 if draft is None else draft.stride(0),
                           target.element_size() * 8, V, u, u_next, B, path, most, n_path, nxt)
    got = path.cpu().numpy(), n_path.tolist(), nxt.tolist()
    t, d = target.double().cpu().numpy()[:, :V], None if draft is None else draft.double().cpu().numpy()[:, :V]
    hu, hn = u.double().cpu().numpy(), u_next.double().cpu().numpy()
    for b in range(B):
        a, z = start[b], start[b + 1]
        want, w_next = orc.verify(parents[a:z], token[a:z], t[a:z], None if d is None else d[a:z], hu[a:z], hn[b], most)
        assert got[1][b] == len(want) and got[0][b][:len(want)].tolist() == want and (got[0][b][len(want):] == -9).all(), b
        assert got[2][b] == w_next, b
    assert got[1][B] == -9 and got[2][B] == -9 and (got[0][B] == -9).all()
    return got


def drafted(seed, B, T, V, dtype, given, shape, pad=0, peak=3.0):
    host, g = random.Random(seed), torch.Generator().manual_seed(seed)
    counts = [host.randint(1, T) for _ in range(B)]
    parents = [p for n in counts for p in [-1] + [j - 1 if shape == "chain" else host.randrange(max(0, j - 3), j) for j in range(1, n)]]
    N = len(parents)
    logits = torch.randn((N, V), generator=g) * peak
    rows = lambda x: torch.nn.functional.pad(torch.softmax(x, 1), (0, pad), value=9.0).to(dtype).to(DEV)
    target, noisy = rows(logits), logits + 0.8 * torch.randn((N, V), generator=g)
    draft = None if given else rows(noisy)
    base = [s for s, n in zip(np.cumsum([0] + counts), counts) for _ in range(n)]
    above = torch.tensor([b + max(p, 0) for b, p in zip(base, parents)])
    p = torch.softmax(noisy, 1)[above]
    token = torch.multinomial(p, 1, generator=g)[:, 0].tolist()
    return counts, parents, token, target, draft, torch.rand(N, generator=g).to(DEV), torch.rand(B, generator=g).to(DEV)


@pytest.mark.parametrize("dtype", [torch.float32, BF])
@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("B, T, V, shape, pad", [
    (1, 6, 32003, "chain", 0), (40, 12, 1000, "tree", 0), (300, 5, 64, "tree", 0), (9, 64, 257, "tree", 3), (3, 9, 100003, "tree", 5),
    (2, 64, 5000, "chain", 0), (150, 4, 9000, "tree", 8), (5, 3, 1, "tree", 0), (1, 2, 1 << 20, "chain", 0)])
def test_verify_against_the_definition(be, dtype, given, B, T, V, shape, pad):
    case = drafted(B * 100 + T + V, B, T, V, dtype, given, shape, pad)
    run_verify(be, *case, most=max(case[0]), vocab=V)


@pytest.mark.parametrize("given", [False, True])
def test_verify_limits_and_odd_numbers(be, given):
    """A path that has no more room, empty sequences, tokens drafted twice, random numbers at and past the ends of their range."""
    host = random.Random(31 + given)
    counts = [0, 7, 0, 8, 5, 6, 8, 0]
    parents = [p for n in counts for p in [-1] + [host.randrange(0, j) for j in range(1, n)] if n]
    N, V = len(parents), 12
    g = torch.Generator().manual_seed(7)
    for round_ in range(40):
        target = torch.softmax(torch.randn((N, V), generator=g) * 2, 1)
        draft = None if given else torch.softmax(torch.randn((N, V), generator=g) * 2, 1).to(DEV)
        token = [host.randrange(-1, 4) for _ in range(N)]
        u = torch.rand(N, generator=g)
        u[round_ % N] = (0.0, 1.0, 2.0, math.nan, -1.0)[round_ % 5]
        un = torch.rand(len(counts), generator=g)
        un[3], un[4] = (0.0, 1.0, math.nan, 0.999999)[round_ % 4], -0.5
        run_verify(be, counts, parents, token, target.to(DEV), draft, u.to(DEV), un.to(DEV), most=3)


@pytest.mark.parametrize("given", [False, True])
def test_verify_probabilities_that_are_none(be, given):
    """Zero rows, NaN, infinities and negative numbers, p equal to q, mass that a rejection uses up, parents that do not exist."""
    inf, nan = math.inf, math.nan
    rows = [[0, 0, 0, 0], [nan, inf, -1, -inf], [1, 0, 0, 0], [0.25] * 4, [nan, 0.5, 0.5, inf], [0, 0, 1e-40, 0], [0.5, 0.5, 0, 0], [0, 1, 0, nan]]
    for seed in range(60):
        host = random.Random(seed)
        counts = [4, 6, 3]
        parents = [-1, 0, 0, 0, -1, 0, 0, 2, 2, 3, -1, 0, host.choice((0, 2, -1, 5, -7))]
        N = len(parents)
        target = torch.tensor([host.choice(rows) for _ in range(N)], device=DEV)
        draft = None if given else torch.tensor([host.choice(rows) for _ in range(N)], device=DEV)
        if not given and seed % 3 == 0:
            draft = target.clone()
        run_verify(be, counts, parents, [host.randrange(-2, 6) for _ in range(N)], target, draft,
                   torch.tensor([host.random() for _ in range(N)], device=DEV), torch.tensor([host.random() for _ in range(3)], device=DEV), most=6)


def test_verify_rows_off_16_bytes(be):
    for dtype, off in ((torch.float32, 1), (BF, 3)):
        counts, parents, token, target, draft, u, un = drafted(77, 4, 6, 4099, dtype, False, "tree", 4)
        t, d = (torch.cat((torch.zeros(off, dtype=dtype, device=DEV), x.reshape(-1)))[off:].view(x.shape) for x in (target, draft))
        assert t.data_ptr() % 16
        run_verify(be, counts, parents, token, t, d, u, un, most=6, vocab=4099)


@pytest.mark.parametrize("given", [False, True])
def test_verify_leaves_the_targets_distribution(be, given):
    """What comes out behind node 0, over 60,000 sequences with random numbers of their own, is distributed as the target's row. A
    share of n draws has a deviation of sqrt(p (1 - p) / n); six of them are allowed."""
    B, V = 60000, 5
    g = torch.Generator(device=DEV).manual_seed(5)
    p = torch.tensor([0.4, 0.3, 0.2, 0.1, 0.0], device=DEV)
    q = torch.tensor([0.1, 0.5, 0.1, 0.2, 0.1], device=DEV)
    target, draft = p.expand(3 * B, V).contiguous(), q.expand(3 * B, V).contiguous()
    token = torch.multinomial(q, 3 * B, replacement=True, generator=g).int() if not given else i32([0, 1, 2]).repeat(B)
    path, n_path, nxt = torch.zeros((B, 3), dtype=torch.int32, device=DEV), i32([0] * B), i32([0] * B)
    be.launch_draft_verify(3 * torch.arange(B + 1, device=DEV).int(), i32([-1, 0, 0]).repeat(B), token, target, V, None if given else draft, V, 32, V,
                           torch.rand(3 * B, device=DEV, generator=g), torch.rand(B, device=DEV, generator=g), B, path, 3, n_path, nxt)
    at = 3 * torch.arange(B, device=DEV) + path[:, 1]
    first = torch.where(n_path > 1, token[at.clamp(0, 3 * B - 1)], nxt)
    share = torch.bincount(first.long(), minlength=V).double() / B
    assert ((share - p).abs() <= 6 * (p * (1 - p) / B).sqrt() + 1e-12).all()
    assert (n_path > 1).double().mean() > 0.3


@pytest.mark.parametrize("dtype, V, given", [(torch.float32, 32003, False), (BF, 151552, True), (BF, 5000, False), (torch.float32, 4099, True)])
def test_verify_draws_every_place(be, dtype, V, given):
    """A draw lands where it has to at the borders of loads, runs, chunks and blocks' parts: three neighbours hold all of a row, in
    quarters whose sums are exact, and the random number is a border itself or lies between two."""
    at = sorted({p for c in (4, 8, 32, 128, 256, 512, 1024, 2048, 4096, 8192, 18944, 32768) for k in (1, 2, 3, 5, 7) for p in (c * k - 1, c * k, c * k + 1)
                 if 1 <= p < V - 1} | {1, 2, V - 2, V - 3})
    B = 4 * len(at)
    mid = torch.tensor(at, device=DEV).repeat(4)
    row = torch.arange(B, device=DEV)
    target = torch.zeros((B, V), dtype=dtype, device=DEV)
    for d, w in ((-1, 0.25), (0, 0.5), (1, 0.25)):
        target[row, mid + d] = w
    u_next = torch.tensor([0.0, 0.25, 0.625, 0.75], device=DEV).repeat_interleave(len(at))
    move = torch.tensor([-1, 0, 0, 1], device=DEV).repeat_interleave(len(at))
    path, n_path, nxt = torch.zeros((B, 1), dtype=torch.int32, device=DEV), i32([0] * B), i32([-9] * B)
    be.launch_draft_verify(i32(range(B + 1)), i32([-1] * B), i32([0] * B), target, V, None if given else target, V, dtype.itemsize * 8, V,
                           torch.zeros(B, device=DEV), u_next, B, path, 1, n_path, nxt)
    assert torch.equal(nxt.long(), mid + move)
    assert (n_path == 1).all() and (path == 0).all()


@pytest.mark.parametrize("B", [1, 37, 80, 400])
def test_verify_few_and_many_sequences(be, B):
    """From eight blocks a sequence to one, with rows of a whole number of chunks and with one value more."""
    for V in (16384, 16385):
        case = drafted(B + V, B, 3, V, BF, B % 2 == 0, "tree", 16384 + 8 - V)
        run_verify(be, *case, most=3, vocab=V)


# --- commit -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("page, kvl, rope, hd, layers, B", [(64, 512, 64, 128, 3, 5), (16, 512, 64, 64, 40, 40), (1, 128, 16, 16, 1, 2), (128, 512, 128, 512, 2, 3)])
def test_commit_against_the_definition(be, page, kvl, rope, hd, layers, B):
    host, g = random.Random(page), np.random.RandomState(page)
    lens = [host.randrange(0, 200) for _ in range(B)]
    cache = Cache(page, [n + 64 for n in lens], page, kvl, rope)
    R, W = cache.n_pages * page, kvl + rope
    paths = [sorted([0] + host.sample(range(1, 64), host.choice((0, 1, 4, 9, 30, 63)))) for _ in range(B)]
    paths[0] = list(range(20))                     # a chain: nothing moves
    if B > 2:
        paths[1] = []
        paths[2] = [3, 4, 5]                       # the root itself is gone
    if B > 4:
        paths[3] = [0, 5, 4]                       # not ascending
        cache.table[4, :] = -1                     # not mapped
        paths[4] = [0, 2, 4]
    pools = [[g.randint(0, 256, (R, W)).astype(np.uint8), g.rand(R).astype(np.float32)] +
             ([g.randint(0, 256, (R, hd)).astype(np.uint8), g.rand(R).astype(np.float32)] if l % 3 != 1 else [None, None]) for l in range(layers)]
    dev = [[None if a is None else torch.from_numpy(a).to(DEV) for a in p] for p in pools]
    geom = be.DsaGeom.make(kv_lora=kvl, rope_dim=rope, index_dim=hd, page_tokens=page, max_pages_per_seq=cache.table.shape[1], n_pool_pages=cache.n_pages)
    arr = i32([p + [-5] * (64 - len(p)) for p in paths])
    status, seq_len = i32([0]), i32([-1] * (B + 1))
    be.launch_kv_commit_paged(geom, be.commit_layers(dev), layers, torch.from_numpy(cache.table).to(DEV), i32(lens), arr, 64,
                              i32([len(p) for p in paths]), B, seq_len, status)
    sound = [orc.commit([a for p in pools for a in p if a is not None], cache.table[b], page, cache.n_pages, lens[b], paths[b]) for b in range(B)]
    for p, d in zip(pools, dev):
        for a, t in zip(p, d):
            assert a is None or np.array_equal(a, t.cpu().numpy())
    assert seq_len.tolist() == [lens[b] + len(paths[b]) if sound[b] else -1 for b in range(B)] + [-1]
    assert status.item() == int(not all(sound))


# --- a run of them together -------------------------------------------------------------------------------------------
def make_stack(be, B, H=64, layers=(True, False, True), page=64):
    from rivoli_b200.engine import DsaDecodeStack
    geom = be.DsaGeom.make(n_heads=H, page_tokens=page, max_pages_per_seq=8 * 64 // page, n_pool_pages=B * 8 * 64 // page + 2)
    return DsaDecodeStack(geom, B, list(layers), device=DEV, shuffle_seed=3)


@pytest.mark.parametrize("H, page", [(64, 64), (16, 16)])
def test_a_drafted_step_is_the_steps_of_its_tokens(be, H, page):
    """Append a tree, attend, verify, commit: each accepted node saw what a step of one token sees on a stack that took the accepted
    tokens one at a time, and the caches hold the same bytes afterwards."""
    from rivoli_b200.draft import DraftStep, DraftTree
    B, V = 3, 50
    g = torch.Generator().manual_seed(11)
    bf = lambda *s: torch.randn(s, generator=g).to(BF).to(DEV)
    parents = [[-1, 0, 0, 2, 2, 4], [-1, 0, 1, 2], [-1]]
    tree = DraftTree(parents, device=DEV)
    N, lens = tree.n_nodes, [130, 63, 5]
    a, b = make_stack(be, B, H, page=page), make_stack(be, B, H, page=page)
    for s in (a, b):
        for i, n in enumerate(lens):
            s.pool.reserve(i, n + 8)
        s.upload_block_table()
    for i in range(3):                                       # the prefixes
        rows = bf(sum(lens), 576), bf(sum(lens), 128)
        seq = torch.repeat_interleave(torch.arange(B), torch.tensor(lens)).int().to(DEV)
        pos = torch.cat([torch.arange(n) for n in lens]).int().to(DEV)
        for s in (a, b):
            s.layers[i].append(*rows, pos, seq)
    rope = be.rope_frequencies(64, 10000.0, "yarn", 4.0)
    step = DraftStep(a, 64, rope, "split")
    x = [(bf(N, 576), bf(N, 128), bf(N, H, 576)) for _ in range(3)]
    step.begin(tree, i32(lens))
    rotated = []
    for latent, key, q in x:
        latent, q = latent.clone(), q.clone()
        step.rotate(q[..., 512:], latent[:, 512:])
        rotated.append((latent, key, q))
    outs = [step.layer(i, *rotated[i]).clone() for i in range(3)]
    # accepted: 0, 2, 4, 5 of the first tree, 0 and 1 of the second
    target = torch.full((N, V), 1e-3, device=DEV)
    token = i32([0, 1, 2, 3, 4, 5, 0, 7, 8, 9, 0])
    for node, t in ((0, 2), (2, 4), (4, 5), (5, 33), (6, 7), (7, 44), (10, 45)):
        target[node, t] = 0.9
    path, n_path, nxt = step.verify(token, target, torch.full((N,), 0.5, device=DEV), torch.full((B,), 0.5, device=DEV))
    assert n_path.tolist() == [4, 2, 1] and path[0, :4].tolist() == [0, 2, 4, 5] and path[1, :2].tolist() == [0, 1]
    assert nxt.tolist() == [33, 44, 45]
    seq_len = i32([0] * B)
    step.commit(seq_len)
    step.check_status()
    assert seq_len.tolist() == [134, 65, 6]
    # the same tokens one at a time
    chains = [[0, 2, 4, 5], [6, 7], [10]]
    from rivoli_b200.layer import DsaDecodeLayer
    for k in range(4):
        who = [c[k] if k < len(c) else None for c in chains]
        live = [i for i, w in enumerate(who) if w is not None]
        idx = torch.tensor([who[i] for i in live], device=DEV)
        at = [lens[i] + k for i in live]
        for l in range(3):
            L = b.layers[l]
            latent, key, q = x[l][0][idx].clone(), x[l][1][idx].clone(), x[l][2][idx].clone()
            f = step.inv_freq
            be.launch_rope_rows_bf16(be.rope_vecs(q[..., 512:]), be.rope_vecs(latent[:, 512:]), len(live), i32(at), f, 64, 2, rope[1])
            L.append(latent, key, i32(at), i32(live))
            full = torch.zeros((B, H, 576), dtype=BF, device=DEV)
            full[live] = q
            out = L.attend(full, dense_len=i32([at[live.index(i)] + 1 if i in live else 0 for i in range(B)])).clone()
            for r, i in enumerate(live):
                got, want = outs[l][idx[r]].float(), out[i].float()
                # Rows and queries of unit deviation: scores are off by 2^-8 / sqrt 3 (the root of sum q^2 k^2 is 24, the scale 1 / 24),
                # weights and results by as much again, of two kernels: sqrt(6) 2^-8 / sqrt 3 = 5.5e-3 of the norm, twice that allowed
                assert (got - want).norm() <= 1.1e-2 * want.norm()
    for l in range(3):
        A, C = a.layers[l], b.layers[l]
        table, P = b.pool.block_table(), page
        for i, n in enumerate(seq_len.tolist()):
            rows = torch.tensor([table[i, t // P] * P + t % P for t in range(n)], device=DEV)
            for name, w in (("latent_pool", 576), ("latent_scale", 1), ("index_pool", 128), ("index_scale", 1)):
                assert torch.equal(getattr(A, name).view(-1, w)[rows], getattr(C, name).view(-1, w)[rows]), (l, i, name)


def test_a_drafted_step_captured(be):
    """The whole step in one graph, replayed on other inputs in the same buffers."""
    from rivoli_b200.draft import DraftStep, DraftTree
    B, V, H = 2, 300, 64
    stack = make_stack(be, B, H, (True,))
    for i in range(B):
        stack.pool.reserve(i, 300)
    stack.upload_block_table()
    step, tree = DraftStep(stack, 32, be.rope_frequencies(64)), DraftTree([[-1, 0, 0, 1], [-1, 0]], device=DEV)
    N, g = tree.n_nodes, torch.Generator().manual_seed(1)
    pos, seq_len = i32([100, 200]), i32([0, 0])
    bufs = dict(latent=torch.zeros((N, 576), dtype=BF, device=DEV), key=torch.zeros((N, 128), dtype=BF, device=DEV),
                q=torch.zeros((N, H, 576), dtype=BF, device=DEV), target=torch.zeros((N, V), device=DEV), draft=torch.zeros((N, V), device=DEV),
                u=torch.zeros(N, device=DEV), un=torch.zeros(B, device=DEV))
    token = i32([0, 3, 5, 7, 0, 9])

    def fill(seed):
        g.manual_seed(seed)
        for name in ("latent", "key", "q"):
            bufs[name].copy_(torch.randn(bufs[name].shape, generator=g))
        for name in ("target", "draft"):
            bufs[name].copy_(torch.softmax(torch.randn((N, V), generator=g) * 3, 1))
        bufs["u"].copy_(torch.rand(N, generator=g))
        bufs["un"].copy_(torch.rand(B, generator=g))
        L = stack.layers[0]
        g2 = torch.Generator(device=DEV).manual_seed(seed)
        L.latent_pool.copy_(torch.randint(0, 120, L.latent_pool.shape, generator=g2, device=DEV))
        L.latent_scale.copy_(torch.rand(L.latent_scale.shape, generator=g2, device=DEV) * 0.01)

    def go(stream=None):
        step.begin(tree, pos, stream)
        step.rotate(bufs["q"][..., 512:], bufs["latent"][:, 512:], stream)
        step.layer(0, bufs["latent"], bufs["key"], bufs["q"], None, stream)
        step.verify(token, bufs["target"], bufs["u"], bufs["un"], bufs["draft"], stream)
        step.commit(seq_len, stream)

    state = lambda: [t.clone() for t in (step.out[:N], step.lse[:N], step.n_path, step.next_token, seq_len, stack.layers[0].latent_pool, stack.layers[0].index_scale)]
    want = []
    for seed in (1, 2, 3):
        fill(seed)
        go()
        torch.cuda.synchronize()
        want.append(state())
    fill(1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        go(side)
    for seed, w in zip((1, 2, 3), want):
        fill(seed)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(state(), w))
    step.check_status()


def test_two_calls_at_once(be):
    """Two streams, a scratch each: the same bits as one after the other."""
    host = random.Random(40)
    runs = []
    for k in range(2):
        trees, prefix = [9 + k, 30], [1200, 300 + 50 * k]
        masks = [m for t in trees for m in masks_of(host, t, "tree")]
        runs.append(run_tree(be, Cache(40 + k, [p + t for p, t in zip(prefix, trees)], 64), 64, prefix, trees, masks, seed=k)[:3])
    streams = [torch.cuda.Stream() for _ in runs]
    again = [(torch.zeros_like(o), torch.zeros_like(l)) for o, l, _ in runs]
    torch.cuda.synchronize()
    for _ in range(5):
        for (o, l), (_, _, args), s in zip(again, runs, streams):
            be.launch_mla_tree_attend_paged_bf16(*args[:13], o, l, args[15], s)
    torch.cuda.synchronize()
    for (o, l), (wo, wl, args) in zip(again, runs):
        assert torch.equal(o[:args[12]], wo[:args[12]]) and torch.equal(l[:args[12]], wl[:args[12]])


def test_step_refuses(be):
    from rivoli_b200.draft import DraftStep, DraftTree
    stack = make_stack(be, 2, 64, (True,))
    step = DraftStep(stack, 4)
    with pytest.raises(ValueError):
        step.begin(DraftTree([[-1, 0, 1], [-1, 0]]), i32([0, 0]))
    with pytest.raises(ValueError):
        step.begin(DraftTree([[-1]]), i32([0]))
    step.begin(DraftTree([[-1], [-1]]), i32([0, 0]))
    p = torch.full((2, 8), 0.125, device=DEV)
    u = torch.zeros(2, device=DEV)
    for bad in (dict(target=p.half()), dict(target=p.t()), dict(target=p, draft=p.to(BF)), dict(target=p, draft=p[:, :4])):
        with pytest.raises(ValueError):
            step.verify(i32([0, 0]), bad["target"], u, u, bad.get("draft"))


def test_step_refuses_what_does_not_fit(be):
    """Sizes, types and strides that a kernel would read past."""
    from rivoli_b200.draft import DraftStep, DraftTree
    stack = make_stack(be, 2, 64, (True, True))
    step = DraftStep(stack, 4)
    step.begin(DraftTree([[-1, 0], [-1]]), i32([0, 0]))
    g = stack.layers[0].g
    p, u, tok = torch.full((3, 8), 0.125, device=DEV), torch.zeros(3, device=DEV), i32([0, 0, 0])
    good = dict(token=tok, target=p, u=u, u_next=u[:2])
    for name, bad in (("token", i32([0, 0])), ("token", tok.long()), ("token", i32([0] * 6)[::2]), ("target", p[:2]), ("u", u[:2]), ("u", u.double()),
                      ("u_next", u[:1]), ("u_next", u.to(BF))):
        with pytest.raises(ValueError):
            step.verify(**{**good, name: bad})
    w = g.kv_lora + g.rope_dim
    lat, key, q = (torch.zeros(x, dtype=BF, device=DEV) for x in ((3, w), (3, g.index_dim), (3, g.n_heads, w)))
    good = dict(latent=lat, index_key=key, q=q)
    for name, bad in (("latent", lat[:2]), ("latent", lat.float()), ("latent", torch.zeros((3, 2 * w), dtype=BF, device=DEV)[:, :w]), ("index_key", key[:, :8]),
                      ("q", q[:2]), ("q", q[:, :1]), ("q", q.transpose(0, 1))):
        with pytest.raises(ValueError):
            step.layer(0, **{**good, name: bad})
    rows, n = torch.zeros((2, 4), dtype=torch.int32, device=DEV), i32([0, 0])
    for bad in ((rows[:1], n), (rows, n[:1]), (rows.t(), n), (rows, n.long())):
        with pytest.raises(ValueError):
            step.layer(0, **good, selection=bad)
    with pytest.raises(ValueError):
        step.rotate(q[:2, :, g.kv_lora:])
    with pytest.raises(ValueError):
        step.commit(n[:1])
    with pytest.raises(ValueError):
        step.commit(n.long())
