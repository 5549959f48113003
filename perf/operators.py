"""Drafted tokens over the paged latent cache: the operators of one speculative decoding step, and what is measured of them.

Kinds of cases (``kind``):

* ``rope``    rotary positions of query heads and keys: three pair layouts, part of the head, frequencies scaled for long contexts
* ``tree``    attention of a tree of drafted tokens over each sequence's cached prefix and the tree's own rows
* ``verify``  drafted tokens held against the target's probabilities with given random numbers; the token that follows
* ``commit``  the accepted tokens' cache rows moved to where the sequence goes on, in all layers of a model

``run`` computes the plain form in elementary torch operations; with ``own`` it calls the framework's entry points.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda:0"
KV_LORA, ROPE, INDEX_DIM, NOPE = 512, 64, 128, 192
WIDTH = KV_LORA + ROPE
LAYERS = 78


def rope(rows, heads, seg, width, layout, scaling, factor, far):
    return dict(kind="rope", rows=rows, heads=heads, seg=seg, width=width, layout=layout, scaling=scaling, factor=factor, far=far)


def tree(batch, nodes, lo, hi, heads=64, page=64, top_k=0, shape="tree"):
    return dict(kind="tree", batch=batch, nodes=nodes, lo=lo, hi=hi, heads=heads, page=page, top_k=top_k, shape=shape)


def verify(batch, nodes, vocab, dtype, given, shape):
    return dict(kind="verify", batch=batch, nodes=nodes, vocab=vocab, dtype=dtype, given=given, shape=shape)


def commit(batch, nodes, kept, layers):
    return dict(kind="commit", batch=batch, nodes=nodes, kept=kept, layers=layers)


def listed():
    return [
        # one new token of one user, before its attention
        dict(rope(1, 64, 64, NOPE + ROPE, "split", "yarn", 4.0, 131071), name="rope-1x64"),
        # a prompt
        dict(rope(16381, 64, 64, NOPE + ROPE, "half", "none", 1.0, 16381), name="rope-16381x64"),
        # the smallest call: one short sequence of a 16-head layer with 16-token pages, a chain of five
        dict(tree(1, 5, 257, 257, heads=16, page=16, shape="chain"), name="tree-1x5x257-small"),
        # one interactive user with a long text and a wide tree
        dict(tree(1, 31, 32771, 32771), name="tree-1x31x32771"),
        # a continuously batched server: ragged contexts and ragged trees
        dict(tree(32, 16, 512, 8192), name="tree-32x16xragged"),
        # trees that share their root's selection of 2,048 rows out of long contexts
        dict(tree(16, 8, 24000, 32768, top_k=2048), name="tree-16x8-of-2048"),
        # the largest: wide trees over long contexts
        dict(tree(8, 64, 16384, 16384), name="tree-8x64x16384"),
        # one user, a chain with the draft model's probabilities
        dict(verify(1, 6, 32003, "f32", False, "chain"), name="verify-1x6x32003"),
        # a batch of trees whose tokens were chosen by rank, over a large vocabulary
        dict(verify(128, 12, 151552, "bf16", True, "tree"), name="verify-128x12x151552"),
        # a batch of sampled trees with the draft model's probabilities
        dict(verify(48, 8, 131072, "f32", False, "tree"), name="verify-48x8x131072"),
        # two accepted drafts of one user in the layers of one stage of a model
        dict(commit(1, 8, 3, 13), name="commit-1x3x13"),
        # the accepted rows of a batch in every layer of the 78-layer model
        dict(commit(64, 16, 5, LAYERS), name="commit-64x5x78"),
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(("rope", "tree", "tree", "tree", "verify", "verify", "commit"))
    if kind == "rope":
        seg = rng.choice((20, 48, 64, 64, 128))
        return rope(_log(rng, 1, 8192), rng.choice((1, 8, 16, 64)), seg, seg + rng.choice((0, 4, 64, 192)),
                    rng.choice(("adjacent", "half", "split")), rng.choice(("none", "linear", "ntk", "yarn")),
                    rng.choice((2.0, 4.0, 16.0)), _log(rng, 64, 1 << 20))
    if kind == "tree":
        heads, page = rng.choice(((64, 64), (64, 64), (64, 16), (16, 16)))
        nodes = _log(rng, 1, 64)
        batch = _log(rng, 1, 32)
        hi = _log(rng, 64, max(65, min(65536, 8 * 64 * 16384 // (batch * nodes))))
        lo = hi if rng.random() < 0.3 else _log(rng, max(1, hi // 16), hi)
        return tree(batch, nodes, lo, hi, heads, page, rng.choice((0, 0, 256, 2048)), rng.choice(("tree", "chain")))
    if kind == "verify":
        nodes = _log(rng, 2, 32)
        vocab = _log(rng, 1000, 160000)
        most = max(1, min(128, 128 * 12 * 151552 // (2 * nodes * vocab)))
        return verify(_log(rng, 1, most), nodes, vocab, rng.choice(("f32", "bf16")), rng.random() < 0.5, rng.choice(("tree", "chain")))
    nodes = rng.randint(4, 64)
    return commit(_log(rng, 1, 64), nodes, rng.randint(2, min(6, nodes - 1)), _log(rng, 1, LAYERS))


# --- inputs -------------------------------------------------------------------------------------------------------
class _Rand:
    def __init__(self, seed):
        self.host = random.Random(seed)
        self.gen = torch.Generator(device=DEV)
        self.gen.manual_seed(seed)

    def normal(self, *shape, dtype=torch.float32):
        return torch.randn(shape, generator=self.gen, device=DEV, dtype=dtype)

    def uniform(self, *shape):
        return torch.rand(shape, generator=self.gen, device=DEV)

    def order(self, n):
        return torch.randperm(n, generator=self.gen, device=DEV)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _spread(lo, hi, n):
    return [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)] if n > 1 else [hi]


def _node_counts(case):
    """Nodes of each sequence's tree: from half of ``nodes`` to all of them."""
    return _spread(max(1, (case["nodes"] + 1) // 2), case["nodes"], case["batch"])


def _parents(counts, shape, host):
    """Node 0 is the token decided last; every other node hangs below an earlier one."""
    return [[-1] + [j - 1 if shape == "chain" else max(0, j - 1 - host.randrange(4)) for j in range(1, n)] for n in counts]


def _visible_bits(parents):
    """Bit i of node j: node i is an ancestor of j, or j itself."""
    bits = []
    for j, p in enumerate(parents):
        bits.append((bits[p] if p >= 0 else 0) | 1 << j)
    return [b - (1 << 64) if b >> 63 else b for b in bits]


def _frequencies(case):
    """Angle per position of each pair, in 64 bits, and what the cosines and sines are multiplied by."""
    seg, theta, factor = case["seg"], 10000.0, case["factor"]
    if case["scaling"] == "ntk":
        theta *= factor ** (seg / (seg - 2))
    f = theta ** (-torch.arange(0, seg, 2, dtype=torch.float64) / seg)
    scale = 1.0
    if case["scaling"] == "linear":
        f = f / factor
    if case["scaling"] == "yarn":
        turns = lambda beta: seg * math.log(4096 / (beta * 2 * math.pi)) / (2 * math.log(theta))
        low, high = max(math.floor(turns(32.0)), 0), min(math.ceil(turns(1.0)), seg - 1)
        ramp = ((torch.arange(seg // 2, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
        f = f / factor * ramp + f * (1 - ramp)
        scale = 0.1 * math.log(factor) + 1.0
    return f, scale


def _prepare_rope(case, rnd):
    n, h, seg, w = case["rows"], case["heads"], case["seg"], case["width"]
    f, scale = _frequencies(case)
    pos = [rnd.host.randrange(case["far"]) for _ in range(n)] if n < 1024 else torch.randint(0, case["far"], (n,), generator=rnd.gen, device=DEV).to(torch.int32)
    bf = torch.bfloat16
    return dict(layout=case["layout"], seg=seg, rows=n, inv_freq=f.to(DEV), scale=scale, pos=pos if n >= 1024 else _i32(pos),
                q=rnd.normal(n, h, w, dtype=bf)[..., w - seg:], k=rnd.normal(n, w, dtype=bf)[..., w - seg:],
                q_out=torch.zeros((n, h, seg), dtype=bf, device=DEV), k_out=torch.zeros((n, seg), dtype=bf, device=DEV))


def _fp8_rows(rnd, n, width):
    """Rows as the cache holds them: e4m3 codes with one scale per row."""
    codes, scale = torch.empty((n, width), dtype=torch.uint8, device=DEV), torch.empty(n, device=DEV)
    step = 1 << 17
    for at in range(0, n, step):
        x = rnd.normal(min(step, n - at), width)
        s = x.abs().amax(1) / 448
        codes[at:at + step] = (x / s[:, None]).to(torch.float8_e4m3fn).view(torch.uint8)
        scale[at:at + step] = s
    return codes, scale


def _pages(rnd, lens, page):
    """A block table over a pool with a quarter of its pages free, pages in random order."""
    need = [-(-n // page) for n in lens]
    pool = math.ceil(1.25 * sum(need))
    order = rnd.order(pool).to(torch.int32)
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, pool


def _tree_lengths(case):
    return _spread(case["lo"], case["hi"], case["batch"]), _node_counts(case)


def _prepare_tree(case, rnd):
    lens, counts = _tree_lengths(case)
    rnd.host.shuffle(lens)
    rnd.host.shuffle(counts)
    page, k, H = case["page"], case["top_k"], case["heads"]
    table, pool = _pages(rnd, [n + t for n, t in zip(lens, counts)], page)
    codes, scale = _fp8_rows(rnd, pool * page, WIDTH)
    start = [sum(counts[:b]) for b in range(len(counts) + 1)]
    s = dict(heads=H, page=page, table=table, codes=codes, pool_scale=scale, tree_pos=_i32(lens), start=_i32(start), n_nodes=start[-1],
             batch=case["batch"], most=max(counts), softmax_scale=WIDTH ** -0.5, rows=None,
             mask=torch.tensor([m for p in _parents(counts, case["shape"], rnd.host) for m in _visible_bits(p)], device=DEV),
             q=rnd.normal(start[-1], H, WIDTH, dtype=torch.bfloat16), n_rows=_i32([min(n, k) if k else n for n in lens]),
             longest=max(min(n, k) if k else n for n in lens))
    if k:
        s["rows"] = torch.zeros((len(lens), k), dtype=torch.int32, device=DEV)
        for b, n in enumerate(lens):
            s["rows"][b, :min(n, k)] = rnd.order(n)[:k].sort().values.to(torch.int32)
    if own:
        from rivoli_b200 import backend as be
        s["geom"] = be.DsaGeom.make(n_heads=H, page_tokens=page, top_k=k or 2048, max_pages_per_seq=table.shape[1], n_pool_pages=pool,
                                    softmax_scale=s["softmax_scale"])
        s["out"] = torch.zeros((start[-1], H, KV_LORA), dtype=torch.bfloat16, device=DEV)
        s["lse"] = torch.zeros((start[-1], H), device=DEV)
        s["scratch"] = torch.zeros(be.mla_tree_attend_scratch_bytes(s["geom"], case["batch"], start[-1]), dtype=torch.uint8, device=DEV)
    return s


def _prepare_verify(case, rnd):
    counts, V = _node_counts(case), case["vocab"]
    rnd.host.shuffle(counts)
    start = [sum(counts[:b]) for b in range(len(counts) + 1)]
    parents = _parents(counts, case["shape"], rnd.host)
    N = start[-1]
    dtype = torch.float32 if case["dtype"] == "f32" else torch.bfloat16
    logits = rnd.normal(N, V).mul_(4.0)
    target = torch.softmax(logits, 1).to(dtype)
    row = torch.tensor([a + max(p, 0) for a, ps in zip(start, parents) for p in ps], device=DEV)
    logits.add_(rnd.normal(N, V).mul_(0.7))
    s = dict(start=_i32(start), parent=_i32([p for ps in parents for p in ps]), target=target, draft=None, vocab=V, batch=case["batch"],
             most=max(counts), u=rnd.uniform(N), u_next=rnd.uniform(case["batch"]))
    if case["given"]:
        rank = [sum(p == ps[j] for p in ps[:j]) for ps in parents for j in range(len(ps))]
        best = logits.topk(max(rank) + 1, dim=1).indices
        s["token"] = best[row, torch.tensor(rank, device=DEV)].to(torch.int32)
    else:
        s["draft"] = torch.softmax(logits, 1).to(dtype)
        s["token"] = torch.multinomial(s["draft"].float()[row], 1, generator=rnd.gen)[:, 0].to(torch.int32)
    s["path"] = torch.full((case["batch"], s["most"]), -1, dtype=torch.int32, device=DEV)
    s["n_path"], s["next"] = _i32([0] * case["batch"]), _i32([-1] * case["batch"])
    return s


def _prepare_commit(case, rnd):
    b, L, page = case["batch"], case["layers"], 64
    lens = _spread(1, 2 * page - 1, b)
    rnd.host.shuffle(lens)
    table, pool = _pages(rnd, [n + case["nodes"] for n in lens], page)
    rows = pool * page
    latent, latent_scale = _fp8_rows(rnd, L * rows, WIDTH)
    key, key_scale = _fp8_rows(rnd, L * rows, INDEX_DIM)
    # node 1 is rejected, so that every accepted row behind the root moves
    path = [[0] + sorted(rnd.host.sample(range(2, case["nodes"]), min(case["kept"] - 1, case["nodes"] - 2))) for _ in range(b)]
    s = dict(latent=latent.view(L, rows, WIDTH), latent_scale=latent_scale.view(L, rows), key=key.view(L, rows, INDEX_DIM),
             key_scale=key_scale.view(L, rows), table=table, tree_pos=_i32(lens), path=_i32(path), n_path=_i32([len(p) for p in path]),
             length=_i32([0] * b), batch=b, page=page)
    if own:
        from rivoli_b200 import backend as be
        s["geom"] = be.DsaGeom.make(max_pages_per_seq=table.shape[1], n_pool_pages=pool)
        s["status"] = _i32([0])
        s["layers"] = be.commit_layers([(s["latent"][i], s["latent_scale"][i], s["key"][i], s["key_scale"][i]) for i in range(L)])
    return s


# --- the plain forms ----------------------------------------------------------------------------------------------
def _run_rope(s):
    seg, half = s["seg"], s["seg"] // 2
    angle = s["pos"].double()[:, None] * s["inv_freq"]
    cos, sin = (angle.cos() * s["scale"]).float(), (angle.sin() * s["scale"]).float()

    def turn(x, c, n):
        x = x.float()
        a, b = (x[..., :half], x[..., half:]) if s["layout"] == "half" else (x[..., 0::2], x[..., 1::2])
        y, z = a * c - b * n, a * n + b * c
        y = torch.stack((y, z), -1).flatten(-2) if s["layout"] == "adjacent" else torch.cat((y, z), -1)
        return y.to(torch.bfloat16)

    return dict(q=turn(s["q"], cos[:, None], sin[:, None]), k=turn(s["k"], cos, sin))


def _rows_of(s):
    """Pool rows [B, longest + most] of each sequence's prefix and tree, and which of them exist."""
    j = torch.arange(s["longest"] + s["most"], device=DEV)[None]
    n, t = s["n_rows"].long()[:, None], (s["start"][1:] - s["start"][:-1]).long()[:, None]
    token = j.expand(s["batch"], -1)
    if s["rows"] is not None:
        token = s["rows"].long().gather(1, j.clamp(max=s["rows"].shape[1] - 1).expand(s["batch"], -1))
    live = j < n + t
    token = torch.where(j < n, token, s["tree_pos"].long()[:, None] + j - n) * live
    return s["table"].long().gather(1, token // s["page"]) * s["page"] + token % s["page"], live, j - n


def _run_tree(s):
    row, live, node = _rows_of(s)
    start = s["start"].long()
    counts = start[1:] - start[:-1]
    t = torch.arange(s["most"], device=DEV)[None]
    there = t < counts[:, None]
    at = (start[:-1, None] + t).clamp(max=s["n_nodes"] - 1)
    k = s["codes"][row].view(torch.float8_e4m3fn).float() * s["pool_scale"][row][..., None]
    bit = (s["mask"][at][..., None] >> node.clamp(0, 63)[:, None]) & 1
    seen = live[:, None] & ((node < 0)[:, None] | (bit > 0))
    q = s["q"][at].float()
    score = torch.einsum("bthd,bld->bthl", q, k) * s["softmax_scale"]
    score = score.masked_fill(~seen[:, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    w = torch.exp(score - torch.where(top > -math.inf, top, 0.0))
    total = w.sum(-1, keepdim=True)
    out = torch.einsum("bthl,bld->bthd", w, k[..., :KV_LORA]) / torch.where(total > 0, total, 1.0)
    lse = (top + total.log())[..., 0]
    return dict(out=out[there].to(torch.bfloat16), lse=lse[there])


def _run_verify(s):
    start, n = s["start"].long(), (s["start"][1:] - s["start"][:-1]).long()
    clean = lambda x: torch.where((x > 0) & (x < math.inf), x, 0.0).double()
    b = torch.arange(s["batch"], device=DEV)
    root = start[:-1]
    cur, r = torch.zeros_like(root), clean(s["target"][root])
    given = s["draft"] is None
    q = None if given else clean(s["draft"][root])
    path, n_path = torch.full_like(s["path"], -1), torch.ones_like(root)
    path[:, 0] = 0
    for j in range(1, s["most"]):
        node = torch.where(j < n, root + j, root)
        x = s["token"][node].long()
        child = (j < n) & (s["parent"][node] == cur)
        qx = 1.0 if given else q[b, x]
        taken = child & (s["u"][node].double() * qx < r[b, x])
        rest = r.clone() if given else (r - q).clamp_(min=0)
        if given:
            rest[b, x] = 0.0
        total = rest.sum(1, keepdim=True)
        rest = torch.where(total > 0, rest / total, 0.0)
        r = torch.where((child & ~taken)[:, None], rest, r)
        r = torch.where(taken[:, None], clean(s["target"][node]), r)
        if not given:
            q = torch.where(taken[:, None], clean(s["draft"][node]), q)
        cur = torch.where(taken, j, cur)
        path[b, n_path.clamp(max=s["most"] - 1)] = torch.where(taken, j, path[b, n_path.clamp(max=s["most"] - 1)].long()).int()
        n_path = n_path + taken
    r = torch.where(r.sum(1, keepdim=True) > 0, r, clean(s["target"][root + cur]))
    cum = r.cumsum(1)
    over = cum > s["u_next"].double()[:, None] * r.sum(1, keepdim=True)
    place = torch.arange(s["vocab"], device=DEV)
    first = torch.where(over & (r > 0), place, s["vocab"]).amin(1)
    last = torch.where(r > 0, place, -1).amax(1)
    return dict(path=path, n_path=n_path.int(), next=torch.where(first < s["vocab"], first, last).int())


def _run_commit(s):
    k = torch.arange(s["path"].shape[1], device=DEV)[None]
    keep = k < s["n_path"][:, None]

    def row(token):
        return (s["table"].long().gather(1, token // s["page"]) * s["page"] + token % s["page"])[keep]

    src, dst = row((s["tree_pos"][:, None] + s["path"]).long()), row((s["tree_pos"][:, None] + k).long())
    for name in ("latent", "latent_scale", "key", "key_scale"):
        s[name][:, dst] = s[name][:, src]
    s["length"].copy_(s["tree_pos"] + s["n_path"])
    return _committed(s)


def _committed(s):
    e4m3 = torch.float8_e4m3fn
    return dict(latent=s["latent"].view(e4m3), latent_scale=s["latent_scale"], key=s["key"].view(e4m3), key_scale=s["key_scale"], length=s["length"])


# --- the framework's operators --------------------------------------------------------------------------------------
def _own_rope(s):
    from rivoli_b200 import backend as be
    be.launch_rope_rows_bf16(be.rope_vecs(s["q"], s["q_out"]), be.rope_vecs(s["k"], s["k_out"]), s["rows"], s["pos"], s["inv_freq"],
                             s["seg"], be.ROPE_LAYOUTS[s["layout"]], s["scale"])
    return dict(q=s["q_out"], k=s["k_out"])


def _own_tree(s):
    from rivoli_b200 import backend as be
    be.launch_mla_tree_attend_paged_bf16(s["geom"], s["q"], s["codes"], s["pool_scale"], s["table"], s["rows"],
                                         0 if s["rows"] is None else s["rows"].shape[1], s["n_rows"], s["tree_pos"], s["start"], s["mask"],
                                         s["batch"], s["n_nodes"], s["out"], s["lse"], s["scratch"])
    return dict(out=s["out"], lse=s["lse"])


def _own_verify(s):
    from rivoli_b200 import backend as be
    t, d = s["target"], s["draft"]
    be.launch_draft_verify(s["start"], s["parent"], s["token"], t, t.stride(0), d, 0 if d is None else d.stride(0), t.element_size() * 8,
                           s["vocab"], s["u"], s["u_next"], s["batch"], s["path"], s["most"], s["n_path"], s["next"])
    return dict(path=s["path"], n_path=s["n_path"], next=s["next"])


def _own_commit(s):
    from rivoli_b200 import backend as be
    be.launch_kv_commit_paged(s["geom"], s["layers"], s["layers"].shape[0], s["table"], s["tree_pos"], s["path"], s["path"].shape[1],
                              s["n_path"], s["batch"], s["length"], s["status"])
    return _committed(s)


_PREPARE = dict(rope=_prepare_rope, tree=_prepare_tree, verify=_prepare_verify, commit=_prepare_commit)
_RUN = dict(rope=_run_rope, tree=_run_tree, verify=_run_verify, commit=_run_commit)
_OWN = dict(rope=_own_rope, tree=_own_tree, verify=_own_verify, commit=_own_commit)


def prepare(case: dict, seed: int):
    s = _PREPARE[case["kind"]](case, _Rand(seed))
    s["kind"] = case["kind"]
    return s


def run(s):
    return _OWN[s["kind"]](s) if own else _RUN[s["kind"]](s)


# --- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "rope":
        vectors = case["rows"] * (case["heads"] + 1)
        return {"bytes": vectors * case["seg"] * 4 + case["rows"] * 4, "flops": vectors * case["seg"] * 3}
    if kind == "tree":
        lens, counts = _tree_lengths(case)
        # the dealing of lengths to trees goes by the seed: the mean over all dealings
        rows = [min(n, case["top_k"]) if case["top_k"] else n for n in lens]
        mean_rows, nodes, H = sum(rows) / len(rows), sum(counts), case["heads"]
        nbytes = (sum(rows) + nodes) * (WIDTH + 4) + nodes * H * (WIDTH * 2 + KV_LORA * 2 + 4)
        return {"bytes": nbytes, "flops": 2 * H * nodes * mean_rows * (WIDTH + KV_LORA)}
    if kind == "verify":
        # the row of probabilities that the next token is drawn from, and the draft's beside it
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": case["batch"] * case["vocab"] * size * (1 if case["given"] else 2) + sum(_node_counts(case)) * 16, "flops": 0}
    moved = case["batch"] * case["layers"] * min(case["kept"] - 1, case["nodes"] - 2)
    return {"bytes": 2 * moved * (WIDTH + INDEX_DIM + 8), "flops": 0}


# --- the definitions in 64 bits ---------------------------------------------------------------------------------------
def _exact_rope(case, s):
    n = case["rows"]
    two_pi = 2 * math.pi
    out = {}
    for name, x in (("q", s["q"].double()), ("k", s["k"].double()[:, None])):
        y = torch.empty_like(x)
        for i, f in enumerate(s["inv_freq"].tolist()):
            a = torch.remainder(s["pos"].double() * f, two_pi)[:, None]
            u, v = (i, i + case["seg"] // 2) if case["layout"] == "half" else (2 * i, 2 * i + 1)
            to = (2 * i, 2 * i + 1) if case["layout"] == "adjacent" else (i, i + case["seg"] // 2)
            y[..., to[0]] = s["scale"] * (x[..., u] * torch.cos(a) - x[..., v] * torch.sin(a))
            y[..., to[1]] = s["scale"] * (x[..., u] * torch.sin(a) + x[..., v] * torch.cos(a))
        out[name] = y if name == "q" else y.view(n, -1)
    return out


def _exact_tree(case, s):
    out, lse = [], []
    start, pos, n_rows, mask = s["start"].tolist(), s["tree_pos"].tolist(), s["n_rows"].tolist(), s["mask"].tolist()
    for b in range(case["batch"]):
        t, n = start[b + 1] - start[b], n_rows[b]
        token = torch.arange(n, device=DEV) if s["rows"] is None else s["rows"][b, :n].long()
        token = torch.cat((token, pos[b] + torch.arange(t, device=DEV)))
        row = s["table"][b].long()[token // case["page"]] * case["page"] + token % case["page"]
        k = s["codes"][row].view(torch.float8_e4m3fn).double() * s["pool_scale"][row].double()[:, None]
        for j in range(t):
            m = mask[start[b] + j]
            hide = [n + i for i in range(t) if not (m >> i) & 1]
            score = s["q"][start[b] + j].double() @ k.T * s["softmax_scale"]
            score[:, hide] = -math.inf
            lse.append(torch.logsumexp(score, 1))
            out.append(torch.exp(score - lse[-1][:, None]) @ k[:, :KV_LORA])
    return dict(out=torch.stack(out), lse=torch.stack(lse))


def _exact_verify(case, s):
    start, parent, token, u, u_next = (s[k].tolist() for k in ("start", "parent", "token", "u", "u_next"))
    path, lengths, following = torch.full((case["batch"], s["most"]), -1, dtype=torch.int32), [], []
    for b in range(case["batch"]):
        a, z = start[b], start[b + 1]
        way = [0]
        while True:
            at = a + way[-1]
            r = s["target"][at].double()
            hit = None
            for j in [j for j in range(1, z - a) if parent[a + j] == way[-1]]:
                x = token[a + j]
                if s["draft"] is None:
                    if u[a + j] < float(r[x]):
                        hit = j
                        break
                    r = r.clone()
                    r[x] = 0
                else:
                    q = s["draft"][at].double()
                    if u[a + j] * float(q[x]) < float(r[x]):
                        hit = j
                        break
                    r = torch.relu(r - q)
                left = float(r.sum())
                r = r / left if left > 0 else r
            if hit is None:
                break
            way.append(hit)
        if float(r.sum()) == 0:
            r = s["target"][a + way[-1]].double()
        over = torch.nonzero(r.cumsum(0) > u_next[b] * r.sum())
        following.append(int(over[0, 0]) if len(over) else int(torch.nonzero(r)[-1, 0]))
        path[b, :len(way)] = torch.tensor(way, dtype=torch.int32)
        lengths.append(len(way))
    return dict(path=path, n_path=torch.tensor(lengths, dtype=torch.int32), next=torch.tensor(following, dtype=torch.int32))


def _exact_commit(case, s):
    out = {n: s[n].view(torch.float8_e4m3fn).double() for n in ("latent", "key")} | {n: s[n].double() for n in ("latent_scale", "key_scale")}
    was = {n: v.clone() for n, v in out.items()}
    table, pos, path, n_path = (s[k].tolist() for k in ("table", "tree_pos", "path", "n_path"))
    place = lambda b, t: table[b][t // s["page"]] * s["page"] + t % s["page"]
    for b in range(case["batch"]):
        for k in range(n_path[b]):
            for n in out:
                out[n][:, place(b, pos[b] + k)] = was[n][:, place(b, pos[b] + path[b][k])]
    return out | {"length": torch.tensor([p + n for p, n in zip(pos, n_path)], dtype=torch.int32)}


def exact(case: dict, seed: int):
    f = dict(rope=_exact_rope, tree=_exact_tree, verify=_exact_verify, commit=_exact_commit)[case["kind"]]
    return f(case, prepare(case, seed))
