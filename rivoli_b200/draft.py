"""A decode step of several drafted tokens per sequence, on the layers of a :class:`~rivoli_b200.engine.DsaDecodeStack`.

The reference decodes one token at a time (``crates/engine/src/glm/decode.rs:128-165``); its caches and calls per layer stay as they
are here (append, then attention), with the trees of all sequences packed into one batch of rows. A step:

    tree = DraftTree(parents)                              # host: which node hangs below which
    step.begin(tree, tree_pos)                             # positions of the step's rows
    per layer:  step.rotate(q, k) ; step.layer(i, ...)     # rotary positions ; append the rows, attend
    step.verify(token, target, u, u_next, draft)           # which nodes stand, and the token that follows
    step.commit(seq_len)                                   # their cache rows to where the sequences go on

Node 0 of a tree is the token decided last, whose cache row this step appends.
"""
from __future__ import annotations

import torch

from . import backend as be

MAX_NODES = 64


def _fits(name: str, t: torch.Tensor, rows: int, shape: tuple, dtype) -> None:
    """At least ``rows`` rows of ``shape``, one behind the other."""
    if t.dim() != len(shape) + 1 or t.shape[0] < rows or tuple(t.shape[1:]) != shape or t.dtype != dtype or not t.is_contiguous():
        raise ValueError(f"{name}: {tuple(t.shape)} of {t.dtype}; contiguous {dtype} of {(rows, *shape)} or more rows")


class DraftTree:
    """The trees of a batch. ``parents[b][j]`` is the node that node ``j`` of sequence ``b`` hangs below, an earlier one; node 0 has
    none (-1). A sequence without nodes sits the step out."""

    def __init__(self, parents: "list[list[int]]", device="cuda:0"):
        start, mask, depth, seq, node = [0], [], [], [], []
        for b, tree in enumerate(parents):
            if len(tree) > MAX_NODES:
                raise ValueError(f"sequence {b}: {len(tree)} nodes, at most {MAX_NODES}")
            bits, deep = [], []
            for j, p in enumerate(tree):
                if (j == 0 and p != -1) or (j > 0 and not 0 <= p < j):
                    raise ValueError(f"sequence {b}: node {j} hangs below {p}")
                bits.append((bits[p] if j else 0) | 1 << j)
                deep.append(deep[p] + 1 if j else 0)
            start.append(start[-1] + len(tree))
            mask += [m - (1 << 64) if m >> 63 else m for m in bits]
            depth += deep
            seq += [b] * len(tree)
            node += range(len(tree))
        if not mask:
            raise ValueError("no nodes")
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)
        self.B, self.n_nodes, self.counts = len(parents), start[-1], [len(t) for t in parents]
        self.max_nodes = max(self.counts)
        self.node_start, self.parent = i32(start), i32([p for t in parents for p in t])
        self.mask = torch.tensor(mask, dtype=torch.int64, device=device)      # u64 payload
        self.depth, self.seq, self.node = i32(depth), i32(seq), i32(node)


class DraftStep:
    """Buffers of the steps of one stack: at most ``max_nodes`` drafted rows a step, all allocated here."""

    def __init__(self, stack, max_nodes: int, rope: "tuple | None" = None, layout: str = "split"):
        """``rope``: what ``backend.rope_frequencies`` gives for the rotated segment, for ``rotate``."""
        L = stack.layers[0]
        g, d, B = L.g, L.dev, L.B
        self.stack, self.max_nodes = stack, max_nodes
        self.out = torch.zeros((max_nodes, g.n_heads, g.kv_lora), dtype=torch.bfloat16, device=d)
        self.lse = torch.zeros((max_nodes, g.n_heads), dtype=torch.float32, device=d)
        self.scratch = torch.zeros(be.mla_tree_attend_scratch_bytes(g, B, max_nodes), dtype=torch.uint8, device=d)
        self.row_pos, self.pos = (torch.zeros(max_nodes, dtype=torch.int32, device=d) for _ in range(2))
        self.tree_pos = torch.zeros(B, dtype=torch.int32, device=d)
        self.path = torch.full((B, MAX_NODES), -1, dtype=torch.int32, device=d)
        self.n_path, self.next_token = (torch.zeros(B, dtype=torch.int32, device=d) for _ in range(2))
        self.pools = be.commit_layers([(K.latent_pool, K.latent_scale, K.index_pool, K.index_scale) for K in stack.layers])
        self.no_key = torch.zeros((max_nodes, g.index_dim), dtype=torch.bfloat16, device=d)   # for layers without an indexer
        self.status = torch.zeros(1, dtype=torch.int32, device=d)
        self.layout = be.ROPE_LAYOUTS[layout]
        self.inv_freq = None if rope is None else torch.as_tensor(rope[0], dtype=torch.float64, device=d).contiguous()
        self.rope_scale = 1.0 if rope is None else rope[1]
        self.tree = None

    def begin(self, tree: DraftTree, tree_pos: torch.Tensor, stream=None) -> None:
        """``tree_pos`` i32 [B]: tokens of each sequence in the cache. The pages of ``tree_pos + nodes`` tokens have to be mapped."""
        if tree.B != self.tree_pos.shape[0] or tree.n_nodes > self.max_nodes:
            raise ValueError(f"{tree.B} trees of {tree.n_nodes} nodes; the step holds {self.tree_pos.shape[0]} of {self.max_nodes}")
        if tree_pos.shape != self.tree_pos.shape or tree_pos.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"tree_pos: {tuple(tree_pos.shape)} of {tree_pos.dtype}; one integer per sequence")
        self.tree, n = tree, tree.n_nodes
        with torch.cuda.stream(be.torch_stream(stream, self.tree_pos.device)):
            self.tree_pos.copy_(tree_pos)
            base = self.tree_pos[tree.seq.long()]
            torch.add(base, tree.node, out=self.row_pos[:n])
            torch.add(base, tree.depth, out=self.pos[:n])

    def rotate(self, q: torch.Tensor, k: "torch.Tensor | None" = None, stream=None) -> None:
        """Rotary positions of the step's rows, in place: ``q`` [n_nodes, heads, seg], ``k`` [n_nodes, seg], views of wider rows."""
        if self.inv_freq is None:
            raise ValueError("rotate: a step without frequencies")
        seg, n = 2 * len(self.inv_freq), self.tree.n_nodes
        for name, t in (("q", q), ("k", k)):
            if t is not None and (t.dim() not in (2, 3) or t.shape[0] < n or t.shape[-1] != seg):
                raise ValueError(f"rotate: {name} of {tuple(t.shape)}; {n} or more rows, segments of {seg}")
        be.launch_rope_rows_bf16(be.rope_vecs(q), None if k is None else be.rope_vecs(k), self.tree.n_nodes, self.pos, self.inv_freq,
                                 q.shape[-1], self.layout, self.rope_scale, stream)

    def layer(self, i: int, latent: torch.Tensor, index_key: "torch.Tensor | None", q: torch.Tensor, selection=None,
              stream=None) -> torch.Tensor:
        """Rows of layer ``i`` into its cache and attention of the tree: ``latent`` [n_nodes, kv_lora + rope], ``index_key``
        [n_nodes, index_dim] or None, ``q`` [n_nodes, heads, kv_lora + rope]. Every node sees the whole prefix, or, with ``selection`` (rows u32
        [B, k], counts i32 [B]), those rows of it: the root's, say, in whose place deeper nodes would have selected their own. Returns
        [n_nodes, heads, kv_lora], a buffer that the next layer writes again."""
        L, t, n = self.stack.layers[i], self.tree, self.tree.n_nodes
        g, bf16 = L.g, torch.bfloat16
        _fits("latent", latent, n, (g.kv_lora + g.rope_dim,), bf16)
        _fits("q", q, n, (g.n_heads, g.kv_lora + g.rope_dim), bf16)
        if index_key is not None:
            _fits("index_key", index_key, n, (g.index_dim,), bf16)
        rows, counts = (None, None) if selection is None else selection
        if rows is not None:
            if rows.dim() != 2 or rows.shape[0] < t.B or rows.dtype not in (torch.int32, torch.uint32) or not rows.is_contiguous():
                raise ValueError(f"selection: {tuple(rows.shape)} of {rows.dtype}; contiguous u32 of {t.B} sequences")
            _fits("selection's counts", counts, t.B, (), torch.int32)
        be.launch_kv_append_paged(L.g, latent, self.no_key if index_key is None else index_key, t.seq, self.row_pos, n, L.block_table,
                                  L.latent_pool, L.latent_scale, L.index_pool, L.index_scale, self.status, stream)
        be.launch_mla_tree_attend_paged_bf16(L.g, q, L.latent_pool, L.latent_scale, L.block_table, rows,
                                             0 if rows is None else rows.shape[1], counts, self.tree_pos, t.node_start, t.mask, t.B, n,
                                             self.out, self.lse, self.scratch, stream)
        return self.out[:n]

    def verify(self, token: torch.Tensor, target: torch.Tensor, u: torch.Tensor, u_next: torch.Tensor,
               draft: "torch.Tensor | None" = None, stream=None):
        """``target``, ``draft`` [n_nodes, vocab] f32 or bf16, ``token`` i32 and ``u`` f32 [n_nodes], ``u_next`` f32 [B]. Fills and
        returns ``path``, ``n_path``, ``next_token``."""
        if target.stride(-1) != 1 or (draft is not None and (draft.stride(-1) != 1 or draft.dtype != target.dtype or draft.shape != target.shape)):
            raise ValueError("probabilities: contiguous rows, draft and target alike")
        if target.dtype not in (torch.float32, torch.bfloat16):
            raise ValueError(f"probabilities in {target.dtype}")
        t = self.tree
        if target.dim() != 2 or target.shape[0] < t.n_nodes:
            raise ValueError(f"probabilities of {tuple(target.shape)} for {t.n_nodes} nodes")
        _fits("token", token, t.n_nodes, (), torch.int32)
        _fits("u", u, t.n_nodes, (), torch.float32)
        _fits("u_next", u_next, t.B, (), torch.float32)
        be.launch_draft_verify(t.node_start, t.parent, token, target, target.stride(0), draft, 0 if draft is None else draft.stride(0),
                               target.element_size() * 8, target.shape[1], u, u_next, t.B, self.path, MAX_NODES, self.n_path,
                               self.next_token, stream)
        return self.path, self.n_path, self.next_token

    def commit(self, seq_len: torch.Tensor, stream=None) -> None:
        """The accepted rows of all layers to their places; ``seq_len`` i32 [B] becomes the tokens in the cache."""
        L = self.stack.layers[0]
        _fits("seq_len", seq_len, self.tree.B, (), torch.int32)
        be.launch_kv_commit_paged(L.g, self.pools, len(self.stack.layers), L.block_table, self.tree_pos, self.path, MAX_NODES,
                                  self.n_path, self.tree.B, seq_len, self.status, stream)

    def check_status(self, stream=None) -> None:
        """Raise if a kernel flagged an unmapped page, an unsound path or a wait that gave up since the last check, in the launches of
        ``stream`` so far (synchronises it)."""
        be.mla_tree_attend_status(self.stack.layers[0].g, self.scratch, stream)
        with torch.cuda.stream(be.torch_stream(stream, self.status.device)):
            flagged = int(self.status.item())
            if flagged:
                self.status.zero_()
        if flagged:
            raise be.BackendError("draft_step(status)", 1005)
