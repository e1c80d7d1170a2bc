"""What the binding of the operators around the MoE layer refuses by itself, on a
CPU-only host: an operator of "cuda:-1" takes CPU tensors as its own, and the
library turns every call that reaches it down for the missing device."""
import pytest

import llmoc_b200 as L

torch = pytest.importorskip("torch")


class Elsewhere:
    """A tensor on another device."""

    def __init__(self, t, device):
        self.t, self.index = t, device

    def __getattr__(self, name):
        return getattr(self.t, name)

    @property
    def device(self):
        return torch.device("cuda", self.index)

    def get_device(self):
        return self.index


def select(ws, ws_bytes):
    bs = L.BeamSearch(1, 4, 64, 4, device=-1)
    i = torch.zeros((1, 4), dtype=torch.int32)
    bs.select(torch.zeros((4, 64)), torch.zeros((1, 4)), i, i.clone(), torch.zeros((1, 4)), ws, ws_bytes)


def test_selection_checks_its_workspace():
    n = L.BeamSearch(1, 4, 64, 4).workspace_bytes()
    ws = torch.empty((n,), dtype=torch.uint8)
    for good in (ws, torch.empty((n // 4,)), ws.data_ptr()):  # stop at the device
        with pytest.raises(L.LlmocError, match="no such CUDA device"):
            select(good, n)
    with pytest.raises(L.LlmocError, match="workspace is on cuda:1"):
        select(Elsewhere(ws, 1), n)
    for bad in (ws[:-1], torch.empty((2 * n,), dtype=torch.uint8)[::2]):
        with pytest.raises(L.LlmocError, match="workspace is no contiguous"):
            select(bad, n)
    with pytest.raises(L.LlmocError, match="workspace too small"):
        select(ws[:-1], n - 1)


def test_moe_block_checks_its_norms_and_workspace():
    """The layer has no handle: what reaches the library is turned down there."""
    layer = L.MoeLayer(None, None, device=-1)
    here, there = L.ResidualNorm(64, pre="rms", device=-1), L.ResidualNorm(64, pre="rms", device=1)
    x = torch.zeros((4, 64), dtype=torch.bfloat16)
    ws = torch.empty((1 << 16,), dtype=torch.uint8)

    def block(before, after, ws, ws_bytes):
        layer.forward_block(before, after, 4, x, x.clone(), x.clone(), ws, ws_bytes)

    for good in (ws, ws.data_ptr()):
        with pytest.raises(L.LlmocError, match="bad arguments"):
            block(here, here, good, ws.numel())
    for norms in ((there, here), (here, there), (there, there)):
        with pytest.raises(L.LlmocError, match="a norm on cuda:1"):
            block(*norms, ws, ws.numel())
    with pytest.raises(L.LlmocError, match="workspace is on cuda:1"):
        block(here, here, Elsewhere(ws, 1), ws.numel())
    with pytest.raises(L.LlmocError, match="workspace is no contiguous"):
        block(here, here, ws, ws.numel() + 1)


def test_reorder_of_a_used_length_changes_all_tensors_or_none():
    a, b = torch.zeros((2, 3, 10, 4)), torch.zeros((2, 3, 6, 4))
    move = L.BeamReorder([a, b], [a.clone(), b.clone()], 2, 3, 3, device=-1, used=5)
    want = [(t.n_seg, t.seg_stride, t.seg_bytes) for t in move.tensors]
    assert want == [(1, 160, 80), (1, 96, 80)]
    for used in (8, -1):  # more than b has
        with pytest.raises(L.LlmocError, match=f"{used} of dimension 0"):
            move.set_used(used)
        assert [(t.n_seg, t.seg_stride, t.seg_bytes) for t in move.tensors] == want


def test_reorder_of_a_used_length_needs_rows_of_one_shape():
    """Rows of other dimensions hold the used part elsewhere; whole rows move as bytes."""
    src, other = torch.zeros((2, 3, 10, 4)), torch.zeros((2, 3, 4, 10))
    L.BeamReorder([src], [other], 2, 3, 3, device=-1)
    L.BeamReorder([src], [torch.zeros((6, 10, 4))], 2, 3, 3, device=-1, dim=1, used=2)  # batch and beams in one
    with pytest.raises(L.LlmocError, match="differ in shape"):
        L.BeamReorder([src], [other], 2, 3, 3, device=-1, used=3)


def test_reorder_refuses_a_dimension_counted_from_the_end():
    """Taken as it is, it would put the end of a row's segment past the row."""
    src = torch.zeros((1, 1, 4, 8))
    for dim in (-1, -2, 2):
        with pytest.raises(L.LlmocError, match=f"dimension {dim}"):
            L.BeamReorder([src], [src.clone()], 1, 1, 1, device=-1, dim=dim, used=3)
