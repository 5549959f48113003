"""The drafted step's operators on the GPU where they can go wrong: long flat tails, rows that are not there, buffers between steps."""
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
