"""Drafted tokens, what needs no GPU: guards of the entry points, the trees, the scaled frequencies, and the 64-bit oracle itself."""
import math

import numpy as np
import pytest
import torch

from oracle import draft_oracle as orc


@pytest.fixture(scope="module")
def be():
    from rivoli_b200 import build
    build.build()
    from rivoli_b200 import backend
    return backend


P = 1 << 20          # an address that nothing reads: a guard refuses first


def refused(be, fn, *args):
    with pytest.raises(be.BackendError) as e:
        fn(*args)
    return e.value.code


def test_rope_guards(be):
    vec = (P, P, 64, 64, 64, 64, 1)
    def code(q=vec, k=None, n=1, pos=P, f=P, seg=64, layout=0):
        return refused(be, be.launch_rope_rows_bf16, q, k, n, pos, f, seg, layout, 1.0)
    assert code(n=0) == 1001 and code(pos=None) == 1001 and code(f=None) == 1001 and code(seg=0) == 1001 and code(q=None) == 1001
    assert code(q=(None, P, 64, 64, 64, 64, 1)) == 1001 and code(q=(P, None, 64, 64, 64, 64, 1)) == 1001 and code(q=(P, P, 0, 0, 0, 0, 0)) == 1001
    assert code(k=(P, P, 64, 64, 64, 64, 0)) == 1001 and code(k=(P, None, 64, 64, 64, 64, 1)) == 1001
    assert code(seg=514) == 1002 and code(q=(P, P, 64, 64, 64, 64, 65537)) == 1002
    assert code(layout=3) == 1003 and code(layout=-1) == 1003
    assert code(seg=63) == 1004
    assert code(q=(P + 1, P, 64, 64, 64, 64, 1)) == 1005 and code(k=(P, P + 1, 64, 64, 64, 64, 1)) == 1005


def test_tree_guards(be):
    G = be.DsaGeom.make(max_pages_per_seq=4, n_pool_pages=8)
    def code(g=G, q=P, rows=None, stride=0, n_rows=P, pos=P, start=P, mask=P, B=1, n=1, out=P, scratch=None, pool=P):
        return refused(be, be.launch_mla_tree_attend_paged_bf16, g, q, pool, P, P, rows, stride, n_rows, pos, start, mask, B, n, out, None, scratch)
    assert code(g=None) == 1001 and code(B=0) == 1001 and code(n=0) == 1001
    for name in ("q", "pos", "start", "mask", "out", "pool"):
        assert code(**{name: None}) == 1001, name
    assert code(rows=P, stride=0) == 1001 and code(rows=P, stride=8, n_rows=None) == 1001
    assert code(n=1 << 24) == 1002 and code(g=be.DsaGeom.make(max_pages_per_seq=4, n_pool_pages=1 << 27)) == 1002
    assert code(g=be.DsaGeom.make(page_tokens=48, max_pages_per_seq=4, n_pool_pages=8)) == 1003
    assert code(g=be.DsaGeom.make(kv_lora=500, max_pages_per_seq=4, n_pool_pages=8)) == 1004
    for name in ("q", "out", "pool", "scratch"):
        assert code(**{name: P + 2}) == 1005, name
    assert code(mask=P + 4) == 1005
    assert be.mla_tree_attend_scratch_bytes(G, 0, 1) == 16


def test_verify_guards(be):
    def code(start=P, parent=P, token=P, target=P, ts=100, draft=None, ds=0, bits=32, vocab=100, u=P, un=P, B=1, path=P, most=8, n=P, nxt=P):
        return refused(be, be.launch_draft_verify, start, parent, token, target, ts, draft, ds, bits, vocab, u, un, B, path, most, n, nxt)
    for name in ("start", "parent", "token", "target", "u", "un", "path", "n", "nxt"):
        assert code(**{name: None}) == 1001, name
    assert code(B=0) == 1001 and code(vocab=0) == 1001 and code(most=0) == 1001
    assert code(vocab=(1 << 20) + 1, ts=1 << 21) == 1002 and code(most=65) == 1002 and code(B=65536) == 1002
    assert code(bits=8) == 1004
    assert code(ts=99) == 1005 and code(draft=P, ds=99) == 1005 and code(target=P + 2) == 1005 and code(target=P + 1, bits=16) == 1005


def test_commit_guards(be):
    G = be.DsaGeom.make(max_pages_per_seq=4, n_pool_pages=8)
    def code(g=G, layers=P, n_layers=1, table=P, pos=P, path=P, stride=8, n=P, B=1, seq_len=None):
        return refused(be, be.launch_kv_commit_paged, g, layers, n_layers, table, pos, path, stride, n, B, seq_len, None)
    for name in ("g", "layers", "table", "pos", "path", "n"):
        assert code(**{name: None}) == 1001, name
    assert code(n_layers=0) == 1001 and code(stride=0) == 1001 and code(B=0) == 1001
    assert code(stride=65) == 1002 and code(B=65536) == 1002
    assert code(layers=P + 4) == 1005 and code(seq_len=P) == 1005


def test_both_ways_of_calling_agree(be):
    """The library's own prototypes, through ctypes, give the codes that the native calls give."""
    L = be.lib()
    assert L.rivoli_rope_rows_bf16(None, None, 1, P, P, 64, 0, 1.0, None) == 1001
    assert L.rivoli_draft_verify(P, P, P, P, 1 << 40, None, 0, 32, 1 << 30, P, P, 1, P, 8, P, P, None) == 1002
    assert L.rivoli_kv_commit_paged(None, P, 1, P, P, P, 8, P, 1, None, None, None) == 1001
    assert L.rivoli_mla_tree_attend_paged_bf16(None, *([P] * 5), 1, *([P] * 4), 1, 1, *([P] * 4)) == 1001
    for name in ("rope_rows_bf16", "draft_verify", "kv_commit_paged", "mla_tree_attend_paged_bf16"):
        with pytest.raises(TypeError):
            getattr(be._launch(), name)(*([None] * (len(be._SIGNATURES[name]) - 1)))


def test_rope_vecs(be):
    x = torch.zeros((3, 4, 96), dtype=torch.bfloat16)
    y = x[..., 32:]
    assert be.rope_vecs(y)[2:] == (384, 96, 384, 96, 4)
    assert be.rope_vecs(x[:, 0, :64], torch.zeros((3, 64), dtype=torch.bfloat16))[2:] == (384, 0, 64, 0, 1)
    for bad in ((x.float(),), (x[..., ::2],), (x, x[..., :64]), (x[0, 0],), (x, x.transpose(0, 1).contiguous().transpose(1, 2))):
        with pytest.raises(ValueError):
            be.rope_vecs(*bad)


@pytest.mark.parametrize("scaling, factor", [("none", 1.0), ("linear", 8.0), ("ntk", 4.0), ("yarn", 16.0)])
def test_frequencies(be, scaling, factor):
    f, scale = be.rope_frequencies(64, 10000.0, scaling, factor)
    plain = 10000.0 ** (-np.arange(32) / 32)
    assert f.dtype == np.float64 and f.shape == (32,) and np.all(np.diff(f) < 0)
    if scaling == "none":
        assert np.allclose(f, plain, rtol=1e-14) and scale == 1.0
    if scaling == "linear":
        assert np.allclose(f, plain / 8, rtol=1e-14) and scale == 1.0
    if scaling == "ntk":                          # the fastest pair as it was, the slowest divided by the factor
        assert f[0] == 1.0 and math.isclose(f[-1], plain[-1] / 4, rel_tol=1e-12) and scale == 1.0
    if scaling == "yarn":                         # pairs that turn often over 4,096 positions as they were, slow ones divided
        turns = plain * 4096 / (2 * math.pi)
        assert np.allclose(f[turns > 40], plain[turns > 40], rtol=1e-12) and np.allclose(f[turns < 0.8], plain[turns < 0.8] / 16, rtol=1e-12)
        assert math.isclose(scale, 0.1 * math.log(16) + 1)


def test_frequencies_refuse(be):
    for args in ((63,), (0,), (64, 1.0), (64, 1e4, "banded"), (64, 1e4, "linear", 0.5), (2, 1e4, "ntk", 2.0)):
        with pytest.raises(ValueError):
            be.rope_frequencies(*args)


def test_trees():
    from rivoli_b200.draft import DraftTree
    t = DraftTree([[-1, 0, 0, 1, 3], [], [-1]], device="cpu")
    assert t.node_start.tolist() == [0, 5, 5, 6] and t.max_nodes == 5 and t.n_nodes == 6 and t.B == 3
    assert t.mask.tolist() == [1, 3, 5, 11, 27, 1] and t.depth.tolist() == [0, 1, 1, 2, 3, 0]
    assert t.seq.tolist() == [0] * 5 + [2] and t.node.tolist() == [0, 1, 2, 3, 4, 0]
    chain = DraftTree([[-1] + list(range(63))], device="cpu")
    assert chain.mask[63] == -1 and chain.mask[62] == (1 << 63) - 1
    for bad in ([[0]], [[-1, 1]], [[-1, -1]], [[-1, 0, 3]], [[-1] * 65], [[]], []):
        with pytest.raises(ValueError):
            DraftTree(bad, device="cpu")


# --- the oracle against what must hold -----------------------------------------------------------------------------
def test_oracle_codes():
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(orc.E4M3, codes, equal_nan=True)


def test_oracle_rope_turns():
    x = np.array([[[1.0, 0.0, 0.0, 2.0]]])
    f = np.array([math.pi / 2, math.pi])
    y = orc.rope(x, np.array([1]), f, "adjacent", 1.0)
    assert np.allclose(y, [[[0, 1, 0, -2]]], atol=1e-12)
    assert np.allclose(orc.rope(x, np.array([1]), f, "split", 3.0), [[[0, 0, 3, -6]]], atol=1e-12)
    z = np.array([[[1.0, 0.0, 0.0, 2.0]]])                  # pairs (1, 0) by a quarter turn, (0, 2) by a half
    assert np.allclose(orc.rope(z, np.array([1]), f, "half", 1.0), [[[0, 0, 1, -2]]], atol=1e-12)
    assert np.allclose(orc.rope(z, np.array([0]), f, "half", 1.0), z)


@pytest.mark.parametrize("given", [False, True])
def test_oracle_verify_leaves_the_targets_distribution(given):
    """Over all values of the random numbers on a fine grid, the token behind node 0 comes out as the target's row says."""
    target = np.array([[0.5, 0.125, 0.375], [1, 0, 0], [1, 0, 0]])
    draft = np.array([[0.25, 0.5, 0.25], [1, 0, 0], [1, 0, 0]])
    grid = (np.arange(16) + 0.5) / 16
    share = np.zeros(3)
    weights = draft[0] if not given else np.array([0.0, 1.0, 0.0])
    for a in range(3):
        for b in range(3):
            w = weights[a] * weights[b] if not given else float((a, b) == (1, 2))
            if not w:
                continue
            for u1 in grid:
                for u2 in grid:
                    for un in grid:
                        path, nxt = orc.verify([-1, 0, 0], [9, a, b], target, None if given else draft, [0, u1, u2], un, 8)
                        share[nxt if len(path) == 1 else (a, b)[path[1] - 1]] += w
    assert np.allclose(share / share.sum(), target[0], atol=0.04)


def test_oracle_verify_edges():
    t = np.array([[0.0, 1.0, 0.0]] * 3)
    assert orc.verify([], [], t, None, [], 0.5, 8) == ([], -1)
    assert orc.verify([-1], [0], t[:1], None, [0], 0.999, 8) == ([0], 1)
    assert orc.verify([-1, 0], [0, 1], t[:2], None, [0, 0.5], 0.5, 8) == ([0, 1], 1)
    assert orc.verify([-1, 0], [0, 1], t[:2], None, [0, 0.5], 0.5, 1) == ([0], 1)       # no room for another node
    assert orc.verify([-1, 0, 0], [0, 0, 1], t, None, [0, 0, 0], 0.5, 8) == ([0, 2], 1)
    assert orc.verify([-1], [0], np.zeros((1, 3)), None, [0], 0.5, 8) == ([0], -1)
    assert orc.verify([-1, 0], [0, 7], t[:2], t[:2], [0, 0], 0.5, 8)[0] == [0]            # no such token


def test_oracle_commit():
    a = np.arange(64, dtype=np.int64)
    assert orc.commit([a], np.array([1, 0]), 16, 2, 14, [0, 2, 3])
    assert a[16 + 15] == 0 and a[0] == 1 and a[1] == 1          # positions 15 and 16 hold what 16 and 17 held
    for path in ([1, 1], [0, 3, 2], [0, 64]):
        assert not orc.commit([a], np.array([1, 0]), 16, 2, 0, path)
    assert not orc.commit([a], np.array([1, -1]), 16, 2, 14, [0, 2])


def test_frequencies_need_an_original_context(be):
    for scaling in ("none", "yarn"):
        with pytest.raises(ValueError):
            be.rope_frequencies(64, 10000.0, scaling, 4.0, 0)


# --- what a step refuses before anything is launched ----------------------------------------------------------------
class Stack:
    """As much of a stack as a step asks for, on the CPU."""

    class pool_layer:
        def __init__(self, be, B):
            self.g, self.dev, self.B = be.DsaGeom.make(n_heads=2, max_pages_per_seq=4, n_pool_pages=8), "cpu", B
            self.latent_pool, self.latent_scale = torch.zeros((512, 576), dtype=torch.uint8), torch.zeros(512)
            self.index_pool, self.index_scale = torch.zeros((512, 128), dtype=torch.uint8), torch.zeros(512)
            self.block_table = torch.zeros((B, 4), dtype=torch.int32)

    def __init__(self, be, B=2, layers=1):
        self.layers = [self.pool_layer(be, B) for _ in range(layers)]


@pytest.fixture()
def step(be, monkeypatch):
    """A step of three nodes in two sequences whose launches are written down instead of made."""
    from rivoli_b200.draft import DraftStep, DraftTree
    s = DraftStep(Stack(be), 4, be.rope_frequencies(64))
    s.tree, s.launched = DraftTree([[-1, 0], [-1]], device="cpu"), []
    for name in ("launch_rope_rows_bf16", "launch_kv_append_paged", "launch_mla_tree_attend_paged_bf16", "launch_draft_verify", "launch_kv_commit_paged"):
        monkeypatch.setattr(be, name, lambda *a, name=name: s.launched.append((name, a)))
    return s


def test_a_step_rotates_keys_of_its_segment_alone(step):
    """A key narrower than the segment would be read and written past its end, a wider one rotated in part."""
    bf = torch.bfloat16
    q, k = torch.zeros((3, 2, 64), dtype=bf), torch.zeros((3, 64), dtype=bf)
    step.rotate(q, k)
    step.rotate(q[:, 0], None)
    assert len(step.launched) == 2
    for bad in (dict(q=q, k=k[:, :32]), dict(q=q, k=torch.zeros((3, 128), dtype=bf)), dict(q=q, k=k[:2]), dict(q=q, k=k[0]), dict(q=q[..., :32], k=k), dict(q=q[:2], k=k)):
        with pytest.raises(ValueError):
            step.rotate(**bad)
    assert len(step.launched) == 2


def test_a_step_keeps_the_key_of_layers_without_one(step):
    """The zero key is one of the step's own buffers: steps of any size, on any stream and captured, read the same one."""
    from rivoli_b200.draft import DraftTree
    bf, keys = torch.bfloat16, []
    for parents in ([[-1, 0], [-1]], [[-1], []], [[-1, 0, 1], [-1]]):
        step.tree = DraftTree(parents, device="cpu")
        step.layer(0, torch.zeros((4, 576), dtype=bf), None, torch.zeros((4, 2, 576), dtype=bf))
        keys.append([a[2] for name, a in step.launched if name == "launch_kv_append_paged"][-1])
    assert keys[0] is keys[1] is keys[2] and any(keys[0] is v for v in vars(step).values())
    assert keys[0].shape == (4, 128) and keys[0].dtype == bf and not keys[0].any()
