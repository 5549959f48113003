"""What the drafted step refuses, without a GPU: types that are not the kernels' own, arrays that overlap."""
import pytest
import torch

from tests.test_draft_host import P, Stack, be, refused, step  # noqa: F401


def test_rope_vecs_of_another_type(be):
    """Two bytes wide is not bf16: halves and integers would be turned as the bf16 that their bits spell."""
    x = torch.zeros((3, 4, 64), dtype=torch.bfloat16)
    be.rope_vecs(x, torch.zeros_like(x))
    for t in (torch.float16, torch.int16):
        for bad in ((x.to(t),), (x, x.to(t)), (x.to(t), x)):
            with pytest.raises(ValueError):
                be.rope_vecs(*bad)


def test_a_selection_of_another_type(step):
    """Rows are 32-bit integers, signed or not: f32 numbers would be read as row numbers by their bits. A step that is refused has not
    written its rows either."""
    bf = torch.bfloat16
    args = torch.zeros((3, 576), dtype=bf), None, torch.zeros((3, 2, 576), dtype=bf)
    rows, n = torch.zeros((2, 4), dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for good in (rows, rows.view(torch.uint32)):
        step.layer(0, *args, selection=(good, n))
    launched = len(step.launched)
    for bad in (rows.float(), rows.long(), rows.short()):
        with pytest.raises(ValueError):
            step.layer(0, *args, selection=(bad, n))
    assert len(step.launched) == launched == 4


def test_a_commit_whose_lengths_overlap_what_it_reads(be):
    """The lengths are written while blocks of other layers still read positions, paths and pages."""
    G, B, stride, far = be.DsaGeom.make(max_pages_per_seq=4, n_pool_pages=8), 3, 8, 1 << 30
    sizes = dict(pos=4 * B, n=4 * B, path=4 * B * stride, table=4 * B * 4)

    def code(seq_len, **at):
        a = {name: far + i * 4096 for i, name in enumerate(sizes)} | at
        return refused(be, be.launch_kv_commit_paged, G, P, 1, a["table"], a["pos"], a["path"], stride, a["n"], B, seq_len, None)

    for name, size in sizes.items():
        for off in (0, 4, size - 4, -4, -(4 * B - 4)):
            assert code(P + off, **{name: P}) == 1005, (name, off)


def test_a_step_begins_with_a_position_per_sequence(step):
    """One position would be given to all sequences, and a fraction cut off."""
    tree, was = step.tree, step.tree_pos.clone()
    for bad in (torch.tensor([5], dtype=torch.int32), torch.tensor(5), torch.tensor([[5, 6]]), torch.tensor([5.5, 6.0]), torch.tensor([5, 6, 7])):
        with pytest.raises(ValueError):
            step.begin(tree, bad)
    assert torch.equal(step.tree_pos, was) and step.tree is tree


def test_rope_segments_written_on_one_another(be):
    """One vector that stands for several is read for each, but not rotated in place once for each, by warps that do not wait for one
    another. (One row, or one vector, may have any stride.)"""
    def code(q, k=None, n=2):
        return refused(be, be.launch_rope_rows_bf16, q, k, n, P, P, 64, 0, 1.0)
    fine = (P, P, 128, 64, 128, 64, 2)
    for bad in ((P, P, 64, 0, 64, 0, 4), (P, P, 0, 64, 0, 64, 4), (P, P, 256, 64, 256, 32, 4), (P, P, 256, 64, 256, -63, 4), (P, P, 64, 64, 63, 64, 1)):
        assert code(bad) == 1005 and code(fine, bad) == 1005, bad
    x = torch.zeros((2, 64), dtype=torch.bfloat16)
    y = x[:, None].expand(2, 4, 64)
    with pytest.raises(be.BackendError):
        be.launch_rope_rows_bf16(be.rope_vecs(y), None, 2, P, P, 64, 0)


def test_a_step_keeps_its_frequencies_in_64_bits(be):
    """Whatever they were given in: the kernel reads eight bytes for each."""
    from rivoli_b200.draft import DraftStep
    f, scale = be.rope_frequencies(64)
    for given in (f, f.astype("f4"), f.tolist(), torch.from_numpy(f), f.repeat(2)[::2]):
        s = DraftStep(Stack(be), 4, (given, scale))
        assert s.inv_freq.dtype == torch.float64 and s.inv_freq.shape == (32,) and s.inv_freq.is_contiguous()
        assert torch.allclose(s.inv_freq, torch.from_numpy(f), rtol=1e-6)


def test_frequencies_of_no_numbers(be):
    """NaN, infinity and turns of zero or fewer gave frequencies that are NaN."""
    nan, inf = float("nan"), float("inf")
    for bad in (dict(theta=nan), dict(theta=inf), dict(factor=nan), dict(factor=inf), dict(original=nan), dict(original=inf), dict(beta_slow=0.0),
                dict(beta_fast=-1.0), dict(beta_fast=nan)):
        with pytest.raises(ValueError):
            be.rope_frequencies(64, **{**dict(theta=10000.0, scaling="yarn", factor=4.0), **bad})
