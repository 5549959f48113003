"""The drafted step's operators on the GPU where they can go wrong: long flat tails, rows that are not there, buffers between steps."""
import math
import random

import numpy as np
import pytest
import torch

from oracle import draft_oracle as orc
from tests.test_draft_gpu import BF, DEV, Cache, be, i32, make_stack, masks_of, signed  # noqa: F401

pytestmark = pytest.mark.gpu


def test_a_captured_step_of_layers_without_a_key(be):
    """Steps of other sizes between two replays take nothing away that the graph reads."""
    from rivoli_b200.draft import DraftStep, DraftTree
    stack = make_stack(be, 2, 16, (True, False))
    for i in range(2):
        stack.pool.reserve(i, 100)
    stack.upload_block_table()
    step, gen = DraftStep(stack, 8), torch.Generator().manual_seed(2)
    trees = [DraftTree(p, device=DEV) for p in ([[-1, 0, 0], [-1]], [[-1], [-1]], [[-1, 0, 1, 2], [-1, 0, 0]])]
    latent, q = (torch.randn(s, generator=gen).to(BF).to(DEV) for s in ((8, 576), (8, 16, 576)))
    pos = i32([30, 64])
    L = stack.layers[1]

    def go(tree, stream=None):
        step.begin(tree, pos, stream)
        step.layer(1, latent, None, q, None, stream)

    def state():
        torch.cuda.synchronize()
        return [t.clone() for t in (step.out[:4], step.lse[:4], L.latent_pool, L.index_pool, L.index_scale)]

    go(trees[0])
    want = state()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        go(trees[0], side)
    for tree in trees[1:]:
        go(tree)
        torch.cuda.synchronize()
        # what the step might have let go of is handed out again
        held = [torch.full((n, 128), 3.0, dtype=BF, device=DEV) for n in (1, 2, 4, 7, 8) for _ in range(4)]
        step.out.zero_(), step.lse.zero_(), L.index_pool.fill_(9), L.latent_pool.fill_(9)
        go(trees[0])
        again = state()
        step.out.zero_(), step.lse.zero_(), L.index_pool.fill_(9), L.latent_pool.fill_(9)
        graph.replay()
        assert all(torch.equal(x, y) for x, y in zip(state(), again))
        del held
    assert all(torch.equal(x, y) for x, y in zip(again[:2], want[:2]))
    step.check_status()


def test_the_status_of_another_stream(be):
    """What a step on a stream of its own flags is seen by a check of that stream, however late the step runs, and is then gone."""
    from rivoli_b200.draft import DraftStep, DraftTree
    stack = make_stack(be, 2, 16, (True,))
    stack.pool.reserve(0, 100)                    # the second sequence has no pages
    stack.upload_block_table()
    step, tree, pos = DraftStep(stack, 4), DraftTree([[-1, 0], [-1]], device=DEV), i32([10, 20])
    latent, key, q = (torch.zeros(s, dtype=BF, device=DEV) for s in ((4, 576), (4, 128), (4, 16, 576)))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)            # some 50 ms
    step.begin(tree, pos, side)
    step.layer(0, latent, key, q, None, side)
    with pytest.raises(be.BackendError):
        step.check_status(side)
    step.check_status(side)
    step.check_status()


@pytest.mark.parametrize("page", [1, 4])
def test_a_commit_whose_rows_are_not_mapped(be, page):
    """Rows that stay where they are have to be there too: a sequence whose pages ran out, or whose position is none, keeps its length."""
    pages = 24 // page
    order = np.random.RandomState(page).permutation(8 * pages).astype(np.int32)
    table = order[:6 * pages].reshape(6, pages).copy()
    pos = [6, 6, 6, 6, -3, 6]
    paths = [[0, 1, 2, 3], [0, 1, 2, 3], [0], [0, 5, 7], [0, 1], [0, 1]]
    table[1, (6 + 3) // page] = -1                # the last of a chain
    table[2, 6 // page] = 8 * pages               # a root alone, past the pool
    table[3, 6 // page] = -1                      # a root that stays before rows that move between pages that are there
    R = 8 * pages * page
    pools = [np.random.RandomState(1).randint(0, 256, (R, 144)).astype(np.uint8), np.random.RandomState(2).rand(R).astype(np.float32)]
    dev = [torch.from_numpy(a).to(DEV) for a in pools]
    geom = be.DsaGeom.make(kv_lora=128, rope_dim=16, index_dim=16, page_tokens=page, max_pages_per_seq=pages, n_pool_pages=8 * pages)
    status, seq_len = i32([0]), i32([-1] * 6)
    arr = i32([p + [-5] * (8 - len(p)) for p in paths])
    be.launch_kv_commit_paged(geom, be.commit_layers([(*dev, None, None)]), 1, torch.from_numpy(table).to(DEV), i32(pos), arr, 8,
                              i32([len(p) for p in paths]), 6, seq_len, status)
    sound = [orc.commit(pools, table[b], page, 8 * pages, pos[b], paths[b]) for b in range(6)]
    assert sound == [True, False, False, False, False, True]
    assert seq_len.tolist() == [10, -1, -1, -1, -1, 8] and status.item() == 1
    assert all(np.array_equal(a, t.cpu().numpy()) for a, t in zip(pools, dev))


@pytest.mark.parametrize("listed", [False, True])
@pytest.mark.parametrize("kvl, page", [(512, 64), (512, 128), (512, 16), (256, 64)])
def test_what_a_row_without_a_scale_holds_does_not_matter(be, kvl, page, listed):
    """NaN codes in rows whose scale is zero or below, anywhere in the prefix and in the tree: the bits that zeros in their place give,
    and what the definition gives without the rows. Tiles of nothing else are among them."""
    host, H, W, n, T = random.Random(page + kvl), 24, kvl + 64, [700, 200], [5, 2]
    cache = Cache(51, [a + b for a, b in zip(n, T)], page, kvl, spread=0.3)
    masks = [m for t in T for m in masks_of(host, t, "tree")]
    lists = [sorted(host.sample(range(m), 150)) for m in n]
    at = [orc.tree_rows(cache.table[b], page, cache.n_pages, 150 if listed else n[b], lists[b] if listed else None, n[b], T[b]) for b in range(2)]
    codes = np.zeros_like(cache.codes)
    for b in range(2):
        dead = set(host.sample(range(len(at[b])), 40)) | ({len(at[b]) - 2} if b == 0 else set()) | (set(range(64, 128)) if b == 0 else set())
        for j in dead:
            cache.scale[at[b][j]] = host.choice((0.0, -1.0))
            codes[at[b][j]] = host.choice((0x7f, 0xff))
            at[b][j] = -1
    nobody = cache.scale <= 0
    cache.codes[nobody] = 0
    g = be.DsaGeom.make(n_heads=H, kv_lora=kvl, page_tokens=page, max_pages_per_seq=cache.table.shape[1], n_pool_pages=cache.n_pages)
    q = torch.randn((7, H, W), generator=torch.Generator().manual_seed(1)).to(BF)
    pool, scale, table = cache.dev()
    sc = torch.zeros(be.mla_tree_attend_scratch_bytes(g, 2, 7), dtype=torch.uint8, device=DEV)
    got = []
    for fill in (False, True):
        if fill:
            rows = torch.from_numpy(nobody).to(DEV)
            pool[rows] = torch.from_numpy(codes).to(DEV)[rows]
        out, lse = torch.zeros((7, H, kvl), dtype=BF, device=DEV), torch.zeros((7, H), device=DEV)
        be.launch_mla_tree_attend_paged_bf16(g, q.to(DEV), pool, scale, table, i32(lists) if listed else None, 150 if listed else 0,
                                             i32([150, 150]) if listed else None, i32(n), i32([0, 5, 7]), signed(masks), 2, 7, out, lse, sc)
        got.append((out, lse))
    be.mla_tree_attend_status(g, sc)
    assert (pool == 0x7f).any() and (pool == 0xff).any()
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    for b, (a, z) in enumerate(((0, 5), (5, 7))):
        want, want_lse = orc.tree_attend(q[a:z].double().numpy(), cache.codes, cache.scale, at[b], 150 if listed else n[b], masks[a:z],
                                         float(np.float32(g.softmax_scale)), kvl)[:2]
        off = got[1][0][a:z].double().cpu().numpy() - want
        # the result's own rounding and the weights' are 2^-8 each at most
        assert np.linalg.norm(off) <= 2.0 ** -7 * np.linalg.norm(want)
        assert np.abs(got[1][1][a:z].double().cpu().numpy() - want_lse).max() <= 2.0 ** -12


# --- long tails under large weights --------------------------------------------------------------------------------------
def behind_a_sink(be, n, B, T, H, page, spread, shares, sink_latent, listed=False, at=0, peaks=0.0):
    """``B`` sequences of ``T`` nodes over one prefix that all of them share: row ``at`` has ``shares[head % ..]`` of the weight, the others
    are flat (``spread`` 0) or have scores of that deviation (every 64th ``peaks`` nats more), and latents with a mean of one in every eighth dim. Returns (out, lse) of
    the call and the definition's (out, lse, sum p |L|) in 64 bits, all [B T, H, ..], and each row's ``shares``."""
    gen = torch.Generator().manual_seed(n + B)
    pages = -(-n // page)
    rows = (pages + B) * page
    x = torch.randn((rows, 576), generator=gen)
    x[:, :512:8] += 1.0
    x[:, 512:] = 0.0
    x[:, 512] = torch.randn(rows, generator=gen) * spread
    x[7::64, 512] += peaks
    x[n:, 512:] = 0.0                                              # rows of the tree score as zero
    x[at, :512] *= sink_latent
    x[at, 512:514] = torch.tensor([0.0, 4.0])
    scale = x.abs().amax(1) / 448
    codes = (x / scale[:, None]).to(torch.float8_e4m3fn).to(DEV)
    k = codes.double() * scale.to(DEV).double()[:, None]
    # scores: the first column's value for all rows but one, for that one what its share asks for
    tail = torch.exp(k[:n, 512]).sum() - math.exp(float(k[at, 512])) + 1.0
    share = torch.tensor([shares[h % len(shares)] for h in range(H)], dtype=torch.float64, device=DEV)
    q = torch.zeros((B * T, H, 576), device=DEV)
    q[..., 512] = 24.0
    q[..., 513] = (24.0 / float(k[at, 513]) * torch.log(share / (1 - share) * tail)).float()
    q = q.to(BF)
    G = be.DsaGeom.make(n_heads=H, page_tokens=page, max_pages_per_seq=pages + 1, n_pool_pages=pages + B)
    table = torch.zeros((B, pages + 1), dtype=torch.int32, device=DEV)
    table[:, :pages] = torch.arange(pages, device=DEV)
    table[:, pages] = pages + torch.arange(B, device=DEV)
    start = i32([T * b for b in range(B + 1)])
    mask = signed([(1 << (j + 1)) - 1 for _ in range(B) for j in range(T)])
    out, lse = torch.zeros((B * T, H, 512), dtype=BF, device=DEV), torch.zeros((B * T, H), device=DEV)
    sc = torch.zeros(be.mla_tree_attend_scratch_bytes(G, B, B * T), dtype=torch.uint8, device=DEV)
    lists = torch.arange(n, dtype=torch.int32, device=DEV).repeat(B, 1) if listed else None
    be.launch_mla_tree_attend_paged_bf16(G, q, codes.view(torch.uint8), scale.to(DEV), table, lists, n if listed else 0, i32([n] * B), i32([pages * page] * B),
                                         start, mask, B, B * T, out, lse, sc)
    be.mla_tree_attend_status(G, sc)
    want = torch.zeros((B * T, H, 512), dtype=torch.float64, device=DEV)
    want_lse, size = torch.zeros((B * T, H), dtype=torch.float64, device=DEV), torch.zeros_like(want)
    for b in range(B):
        for j in range(T):
            own = (pages + b) * page + torch.arange(j + 1, device=DEV)
            at_rows = torch.cat((torch.arange(n, device=DEV), own))
            kk = k[at_rows]
            s = q[b * T + j].double() @ kk.T / 24.0
            top = s.amax(1, keepdim=True)
            p = torch.exp(s - top)
            total = p.sum(1, keepdim=True)
            want_lse[b * T + j] = (top + total.log())[:, 0]
            want[b * T + j], size[b * T + j] = p / total @ kk[:, :512], p / total @ kk[:, :512].abs()
    assert ((torch.exp(s[:, at] - want_lse[-1]) - share).abs() <= 0.05 * (1 - share) + 0.01).all()
    return out.double(), lse.double(), want, want_lse, size, share


SHARES = (0.3, 0.5, 0.9)


@pytest.mark.parametrize("spread", [0.0, 0.5])
@pytest.mark.parametrize("n, page, listed", [(2048, 64, False), (2048, 16, False), (2048, 64, True), (16384, 64, False), (16384, 16, False),
                                             (16384, 64, True), (65536, 64, False)])
def test_a_flat_tail_behind_a_row_with_most_of_the_weight(be, n, spread, page, listed):
    """As many blocks of rows as SMs, each whole in one run. The result's rounding is 2^-8 of an entry at most, the large weight's 2^-9;
    of the others' weights the sum of what rounding takes is held to 2^-11 of all, and 2^-9 in the large one's own tile: 2^-7 of the
    norm together, whatever the length."""
    out, lse, want, want_lse, _, _ = behind_a_sink(be, n, 37, 4, 64, page, spread, SHARES, 1.0, listed)
    off = (out - want).norm(dim=-1) / want.norm(dim=-1)
    assert (off <= 2.0 ** -7).all(), off.max()
    assert (lse - want_lse).abs().max() <= 2.0 ** -14


@pytest.mark.parametrize("n", [16384, 65536])
def test_a_tail_with_peaks_of_its_own(be, n):
    """Every 64th row of the tail is five nats above the others, which have a third of its weight together. Bounds as above."""
    out, lse, want, want_lse, _, _ = behind_a_sink(be, n, 37, 4, 64, 64, 0.0, SHARES, 1.0, peaks=5.0)
    off = (out - want).norm(dim=-1) / want.norm(dim=-1)
    assert (off <= 2.0 ** -7).all(), off.max()
    assert (lse - want_lse).abs().max() <= 2.0 ** -14


@pytest.mark.parametrize("n, share, at, B, T", [
    (32770, 0.5, 0, 37, 4), (32770, 0.931, 0, 37, 4), (32770, 0.99, 0, 1, 1), (16384, 0.9, 9000, 37, 4), (20000, 0.9, 19990, 37, 4), (131072, 0.7, 64, 4, 3)])
def test_a_tail_that_is_the_whole_output(be, n, share, at, B, T):
    """The large weight's own latent is next to nothing, as that of a first token often is: what comes out is the tail. Entries are off by
    2^-8 for the result's rounding and by 2^-9 of sum p |L| for the weights'; 2^-11 of all weights may be lost, of the tail's (1 - share),
    and of the row's own tile 63 rows."""
    out, lse, want, want_lse, size, _ = behind_a_sink(be, n, B, T, 64, 64, 0.0, (share,), 2.0 ** -12, at=at)
    lost = 2.0 ** -11 / (1 - share) + 64.0 / n
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -9 + lost) * size
    assert ((out - want).abs() <= tol).all(), ((out - want).abs() / tol).max()
    assert (lse - want_lse).abs().max() <= 2.0 ** -14


@pytest.mark.parametrize("listed", [False, True])
def test_levels_that_rise_and_fall(be, listed):
    """Stretches of rows tens of binades apart, in both orders, and rows of scales down to 2^-80 among them: references go up and down by
    all of it, sums stay finite, and each row's output is right to the weights' and the result's rounding."""
    n, H, T, page = 8192, 64, 2, 64
    gen = torch.Generator().manual_seed(9)
    rows = n + page
    x = torch.randn((rows, 576), generator=gen)
    x[:, 512:] = 0.0
    scale = x.abs().amax(1) / 448
    level = torch.tensor([0.0, -9.0, -30.0, 4.0, -18.0, -60.0, -12.0, 9.0])      # nats; of stretches of 320 rows
    x[:, 512] = level[(torch.arange(rows) // 320) % 8] * 0.0625
    codes = (x / scale[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    wide = torch.zeros(rows, dtype=torch.int32)
    wide[torch.randperm(n, generator=gen)[:400]] = torch.randint(-80, 1, (400,), generator=gen, dtype=torch.int32)
    scale = torch.ldexp(scale, wide)
    codes, scale = codes.to(DEV), scale.to(DEV)
    k = codes.double() * scale.double()[:, None]
    q = torch.zeros((T, H, 576))
    q[..., 512] = 24.0 * 16 * torch.linspace(-1, 1, H)
    q = q.to(BF).to(DEV)
    G = be.DsaGeom.make(n_heads=H, page_tokens=page, max_pages_per_seq=rows // page, n_pool_pages=rows // page)
    table = torch.arange(rows // page, dtype=torch.int32, device=DEV)[None].contiguous()
    out, lse = torch.zeros((T, H, 512), dtype=BF, device=DEV), torch.zeros((T, H), device=DEV)
    sc = torch.zeros(be.mla_tree_attend_scratch_bytes(G, 1, T), dtype=torch.uint8, device=DEV)
    lists = torch.arange(n, dtype=torch.int32, device=DEV)[None] if listed else None
    be.launch_mla_tree_attend_paged_bf16(G, q, codes.view(torch.uint8), scale, table, lists, n if listed else 0, i32([n]), i32([n]), i32([0, T]), signed([1, 3]),
                                         1, T, out, lse, sc)
    be.mla_tree_attend_status(G, sc)
    for j in range(T):
        kk = k[:n + j + 1]
        s = q[j].double() @ kk.T / 24.0
        lse_j = torch.logsumexp(s, 1)
        p = torch.exp(s - lse_j[:, None])
        want, size = p @ kk[:, :512], p @ kk[:, :512].abs()
        # weights are rounded in units of weight times scale: each of a tile's 64 is off by 2^-15 of the tile's largest such product
        step = torch.nn.functional.pad(p * scale.double()[:n + j + 1], (0, -(n + j + 1) % 64)).view(H, -1, 64).amax(2).sum(1, keepdim=True) * 448
        tol = 2.0 ** -8 * want.abs() + 2.0 ** -8 * size + 2.0 ** -9 * step
        assert out[j].isfinite().all()
        assert ((out[j].double() - want).abs() <= tol).all(), ((out[j].double() - want).abs() / tol).max()
        assert ((lse[j].double() - lse_j).abs() <= 2.0 ** -14 + 2.0 ** -20 * lse_j.abs()).all()


@pytest.mark.parametrize("kvl, page", [(512, 64), (512, 16), (256, 64)])
def test_a_selection_that_names_the_tree(be, kvl, page):
    """The root's selection, made once its row was appended, names that row or counts it: the node sees it once. So with any row from the
    tree's first on, and with no position at all."""
    host, H, n, T = random.Random(61), 16, [300, 90, 200, 128, 40], [3, 2, 4, 1, 2]
    cache = Cache(61, [a + b for a, b in zip(n, T)], page, kvl)
    masks = [m for t in T for m in masks_of(host, t, "tree")]
    k = 160
    rows = [sorted(host.sample(range(m), min(m, k - 4))) for m in n]
    own = [r + [m, m + 1, m + t - 1, 0x80000000 + m][:k - len(r)] for r, m, t in zip(rows, n, T)]
    own = [r + [0] * (k - len(r)) for r in own]
    own[1], own[4] = [0xffffffff] + [0] * (k - 1), [0xffffffff] + [0] * (k - 1)
    counts = [len(r) + 4 for r in rows]
    counts[1], counts[4] = n[1] + 1, 1000                          # dense, with the root counted, and with all that is mapped
    g = be.DsaGeom.make(n_heads=H, kv_lora=kvl, page_tokens=page, max_pages_per_seq=cache.table.shape[1], n_pool_pages=cache.n_pages)
    q = torch.randn((sum(T), H, kvl + 64), generator=torch.Generator().manual_seed(1)).to(BF).to(DEV)
    start = np.concatenate(([0], np.cumsum(T))).tolist()
    pool, scale, table = cache.dev()
    sc = torch.zeros(be.mla_tree_attend_scratch_bytes(g, 5, sum(T)), dtype=torch.uint8, device=DEV)
    got = []
    plain = [r + [0] * (k - len(r)) for r in rows]
    plain[1], plain[4] = own[1], own[4]
    for lists, c in ((plain, [len(rows[0]), n[1], len(rows[2]), len(rows[3]), n[4]]), (own, counts)):
        out, lse = torch.zeros((sum(T), H, kvl), dtype=BF, device=DEV), torch.zeros((sum(T), H), device=DEV)
        r = i32([[v - (1 << 32) if v >> 31 else v for v in row] for row in lists])
        be.launch_mla_tree_attend_paged_bf16(g, q, pool, scale, table, r, k, i32(c), i32(n), i32(start), signed(masks), 5, sum(T), out, lse, sc)
        got.append((out, lse))
    be.mla_tree_attend_status(g, sc)
    # the same rows, but for zeros between them, which shift them to other tiles: sums in another order, weights in other units
    for b in range(5):
        a, z = start[b], start[b + 1]
        x, y = (o[0][a:z].double() for o in got)
        assert (x - y).norm() <= 2.0 ** -8 * x.norm(), b
        assert (got[0][1][a:z] - got[1][1][a:z]).abs().max() <= 2.0 ** -14, b
    nobody = torch.zeros_like(got[0][0]), torch.zeros_like(got[0][1])
    be.launch_mla_tree_attend_paged_bf16(g, q, pool, scale, table, r, k, i32(counts), i32([-5] * 5), i32(start), signed(masks), 5, sum(T), *nobody, sc)
    assert (nobody[0] == 0).all() and (nobody[1] == -math.inf).all()
