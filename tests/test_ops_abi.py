"""The refusals of the operators around the MoE layer, on a CPU-only host:
every call below is turned down by its arguments alone, before any device
work (addresses are made up and never read)."""
import ctypes as C

import pytest

import llmoc_b200 as L

lib = L.lib
A = 1 << 20  # a made-up, well-aligned address; A * n are far apart


def views(n=1, **kw):
    v = dict(q=A, scales=2 * A, zeros=None, M=64, K=128, group_size=64, scheme=2, awq_zp=7)
    v.update(kw)
    return (L.Int4View * n)(*[L.view(**v) for _ in range(n)])


@pytest.mark.parametrize("v,n,code", [
    (views(K=100), 1, 6), (views(group_size=48), 1, 6), (views(K=0), 1, 1), (views(M=0), 1, 1), (views(q=None), 1, 1),
    (views(scales=None), 1, 1), (views(scheme=3), 1, 1), (views(scheme=0), 1, 1), (views(awq_zp=128), 1, 6),
    (views(), 0, 1), (views(2, M=17), 2, 6), (views(3, M=1 << 30), 3, 6), (None, 1, 1),
])
def test_linear_create_refusals(v, n, code):
    h = C.c_void_p(5)
    assert lib.llmoc_int4_linear_create(v, n, 0, 1, C.byref(h)) == code, L.last_error()
    assert h.value is None and L.last_error()


def test_linear_create_refuses_views_that_differ():
    for kw in (dict(K=192), dict(group_size=32), dict(scheme=1), dict(awq_zp=8)):
        v = (L.Int4View * 2)(views()[0], views(**kw)[0])
        h = C.c_void_p()
        assert lib.llmoc_int4_linear_create(v, 2, 0, 1, C.byref(h)) == 1 and "differs" in L.last_error()


def test_linear_null_handle():
    assert lib.llmoc_int4_linear_forward(None, A, 128, 1, None, 0, 2 * A, 64, 0, None) == 1
    assert lib.llmoc_int4_linear_weight_bytes(None) == 0
    lib.llmoc_int4_linear_destroy(None)
    assert lib.llmoc_int4_linear_create(views(), 1, 0, 1, None) == 1


def norm_desc(**kw):
    d = dict(hidden=64, post=1, pre=2, weight_dtype=1, post_weight=A, post_bias=None, pre_weight=2 * A, pre_bias=3 * A,
             weight_offset=0.0, eps=1e-6, block_scale=1.0, residual_scale=1.0, gate_act=0)
    d.update(kw)
    return L.NormDesc(*[d[f[0]] for f in L.NormDesc._fields_])


def norm_io(**kw):
    d = dict(block=10 * A, ld_block=64, residual=11 * A, ld_residual=64, residual_out=12 * A, ld_residual_out=64,
             norm_out=13 * A, ld_norm_out=64, gate=None, gate_row_stride=0, gate_col_stride=0, block_dtype=1,
             residual_dtype=1, norm_dtype=1, gate_dtype=1)
    d.update(kw)
    return L.NormIO(*[d[f[0]] for f in L.NormIO._fields_])


@pytest.mark.parametrize("kw,code", [
    (dict(hidden=0), 1), (dict(hidden=16385), 6), (dict(post=3), 1), (dict(pre=-1), 1), (dict(weight_dtype=2), 1),
    (dict(eps=0.0), 1), (dict(eps=float("nan")), 1), (dict(eps=float("inf")), 1), (dict(gate_act=2), 1),
    (dict(post_weight=A + 1), 1),
])
def test_norm_desc_refusals(kw, code):
    assert lib.llmoc_norm_residual(C.byref(norm_desc(**kw)), C.byref(norm_io()), 4, 0, None) == code, L.last_error()


@pytest.mark.parametrize("kw", [
    dict(block=None, residual=None), dict(residual_out=None, norm_out=None), dict(ld_block=63), dict(ld_norm_out=0),
    dict(block_dtype=2), dict(gate_dtype=-1), dict(block=None, gate=A), dict(gate=20 * A, gate_col_stride=2),
    dict(gate=20 * A, gate_row_stride=-1), dict(norm_out=13 * A + 1), dict(residual_dtype=0, residual=11 * A + 2),
    dict(norm_out=12 * A), dict(norm_out=12 * A + 128), dict(residual_out=11 * A + 128), dict(norm_out=10 * A, norm_dtype=0),
    dict(residual_out=11 * A, ld_residual_out=72), dict(gate=12 * A, gate_row_stride=1),
    dict(gate=13 * A, gate_row_stride=64, gate_col_stride=1),
])
def test_norm_io_refusals(kw):
    assert lib.llmoc_norm_residual(C.byref(norm_desc()), C.byref(norm_io(**kw)), 4, 0, None) == 1, L.last_error()
    assert L.last_error()


def test_norm_empty_batch_and_negative():
    assert lib.llmoc_norm_residual(C.byref(norm_desc()), C.byref(norm_io()), 0, 0, None) == 0
    assert lib.llmoc_norm_residual(C.byref(norm_desc()), C.byref(norm_io()), -1, 0, None) == 1
    assert lib.llmoc_norm_residual(None, C.byref(norm_io()), 1, 0, None) == 1
    assert lib.llmoc_norm_residual(C.byref(norm_desc()), None, 1, 0, None) == 1
    assert lib.llmoc_moe_forward_block(None, C.byref(norm_desc()), C.byref(norm_desc()), C.byref(norm_io()), 1, A, 1 << 30,
                                       None) == 1
    assert lib.llmoc_moe_block_workspace_bytes(None, 4) == 0


def beam(**kw):
    d = dict(batch=2, beams=3, vocab=100, n_out=4, eos_token=-1)
    d.update(kw)
    return L.BeamDesc(*[d[f[0]] for f in L.BeamDesc._fields_])


def select(desc, **kw):
    d = dict(logits=A, ld=100, dtype=1, scores=2 * A, finished=None, parent=3 * A, token=4 * A, out=5 * A, fin_out=6 * A,
             ws=7 * A, ws_bytes=1 << 19, device=0, stream=None)
    d.update(kw)
    return lib.llmoc_beam_select(C.byref(desc), *d.values())


@pytest.mark.parametrize("kw,code", [
    (dict(batch=-1), 1), (dict(beams=0), 1), (dict(vocab=0), 1), (dict(n_out=0), 1), (dict(eos_token=-2), 1),
    (dict(eos_token=100), 1), (dict(beams=129), 6), (dict(n_out=129), 6), (dict(vocab=(1 << 30) + 1), 6),
    (dict(batch=1 << 24), 6),
])
def test_beam_desc_refusals(kw, code):
    d = beam(**kw)
    assert select(d, ld=d.vocab) == code, L.last_error()
    assert lib.llmoc_beam_workspace_bytes(C.byref(d)) == 0


@pytest.mark.parametrize("kw,code", [
    (dict(logits=None), 1), (dict(scores=None), 1), (dict(parent=None), 1), (dict(out=None), 1), (dict(ld=99), 1),
    (dict(dtype=2), 1), (dict(finished=8 * A), 1), (dict(logits=A + 1), 1), (dict(token=4 * A + 2), 1),
    (dict(ws=None), 7), (dict(ws_bytes=64), 7), (dict(ws=7 * A + 4), 1), (dict(parent=2 * A), 1), (dict(token=A), 1),
    (dict(token=3 * A + 16), 1), (dict(fin_out=5 * A + 31), 1),
])
def test_beam_select_refusals(kw, code):
    assert select(beam(), **kw) == code, L.last_error()


def test_beam_empty_batch():
    assert select(beam(batch=0)) == 0


def tensor(**kw):
    d = dict(src=A, dst=2 * A, src_stride=64, dst_stride=64, seg_stride=0, seg_bytes=64, n_seg=1)
    d.update(kw)
    return L.ReorderTensor(*[d[f[0]] for f in L.ReorderTensor._fields_])


@pytest.mark.parametrize("ts", [
    [tensor(src=None)], [tensor(dst=None)], [tensor(n_seg=0)], [tensor(seg_bytes=-1)], [tensor(src_stride=63)],
    [tensor(dst_stride=0)], [tensor(n_seg=2, seg_stride=32, seg_bytes=33, src_stride=100, dst_stride=100)],
    [tensor(n_seg=2, seg_stride=64)], [tensor(n_seg=2, seg_stride=-64)], [tensor(dst=A + 64)],
    [tensor(dst=A, dst_stride=128)], [tensor(), tensor(src=3 * A)], [tensor(), tensor(src=3 * A, dst=A + 511)],
    [tensor(), tensor(src=2 * A, dst=3 * A)], [tensor(src=A, dst=A), tensor(src=A, dst=3 * A)],
])
def test_reorder_refusals(ts):
    arr = (L.ReorderTensor * len(ts))(*ts)
    assert lib.llmoc_beam_reorder(arr, len(ts), 9 * A, 2, 4, 4, 0, None) == 1, L.last_error()
    assert L.last_error()


def test_reorder_shapes():
    t = (L.ReorderTensor * 1)(tensor())
    assert lib.llmoc_beam_reorder(t, 1, None, 2, 4, 4, 0, None) == 1
    assert lib.llmoc_beam_reorder(t, 1, 9 * A + 2, 2, 4, 4, 0, None) == 1
    assert lib.llmoc_beam_reorder(t, 1, 9 * A, 2, 4, 65, 0, None) == 6
    assert lib.llmoc_beam_reorder(t, 1, 9 * A, 1 << 24, 4, 4, 0, None) == 6
    assert lib.llmoc_beam_reorder(t, 1, 9 * A, 2, 0, 4, 0, None) == 1
    assert lib.llmoc_beam_reorder(t, -1, 9 * A, 2, 4, 4, 0, None) == 1
    assert lib.llmoc_beam_reorder(t, 1, 9 * A, 0, 4, 4, 0, None) == 0
    assert lib.llmoc_beam_reorder(None, 0, 9 * A, 2, 4, 4, 0, None) == 0
    # in place with another number of rows: the rows would move under one another
    t = (L.ReorderTensor * 1)(tensor(dst=A))
    assert lib.llmoc_beam_reorder(t, 1, 9 * A, 2, 4, 3, 0, None) == 1


def test_accepted_calls_need_a_device():
    """The same arguments pass every check and stop at the missing device."""
    if lib.llmoc_cuda_probe_available():
        pytest.skip("a GPU is present: the made-up addresses would be used")
    h = C.c_void_p()
    assert lib.llmoc_int4_linear_create(views(2), 2, 0, 1, C.byref(h)) == 2
    assert lib.llmoc_norm_residual(C.byref(norm_desc()), C.byref(norm_io()), 4, 0, None) == 2
    assert lib.llmoc_norm_residual(C.byref(norm_desc()), C.byref(norm_io(residual_out=11 * A, norm_out=10 * A)), 4, 0,
                                   None) == 2
    assert select(beam()) == 2
    assert select(beam(eos_token=3), finished=8 * A) == 2
    t = (L.ReorderTensor * 3)(tensor(), tensor(src=3 * A, dst=3 * A),
                              tensor(src=4 * A, dst=5 * A, n_seg=3, seg_stride=512, src_stride=64, dst_stride=64))
    assert lib.llmoc_beam_reorder(t, 3, 9 * A, 2, 4, 4, 0, None) == 2


def test_linear_status_refuses_a_null_handle():
    assert lib.llmoc_int4_linear_status(None, None) == 1 and "null linear" in L.last_error()


@pytest.mark.parametrize("ws", [A, 2 * A, 3 * A, 4 * A, 5 * A])
def test_beam_workspace_apart_from_operands(ws):
    assert select(beam(), ws=ws) == 1 and "workspace overlaps" in L.last_error()


@pytest.mark.parametrize("beams,vocab", [(1, 500), (4, 32003), (8, 32003), (4, 248320), (8, 248320), (5, 131072),
                                         (128, 70001), (1, 1 << 20), (3, 8192)])
def test_beam_workspace_of_a_batch_serves_smaller_ones(beams, vocab):
    """As sequences end, calls with fewer of them take the workspace that the
    largest batch asked for, with logits of either type."""
    far = 1 << 50
    sizes = [lib.llmoc_beam_workspace_bytes(C.byref(beam(batch=b, beams=beams, vocab=vocab))) for b in range(1, 201)]
    assert sizes == sorted(sizes) and sizes[0] > 0
    big = [1 << i for i in range(8, 25 - beams.bit_length())]
    more = [lib.llmoc_beam_workspace_bytes(C.byref(beam(batch=b, beams=beams, vocab=vocab))) for b in big]
    assert [sizes[-1], *more] == sorted([sizes[-1], *more])
    for dtype in (0, 1):
        for top in (10, 25, 120, 200):
            for b in range(1, top + 1):
                # passes every check and stops at the device, which no machine has
                d = beam(batch=b, beams=beams, vocab=vocab)
                code = select(d, ld=vocab, dtype=dtype, logits=far, scores=2 * far, parent=3 * far, token=4 * far,
                              out=5 * far, fin_out=6 * far, ws=7 * far, ws_bytes=sizes[top - 1], device=1 << 20)
                assert code == 2, (b, top, L.last_error())


def test_beam_workspace_of_the_largest_description():
    """The size is found without walking through millions of batches at length."""
    import time

    t = time.monotonic()
    assert lib.llmoc_beam_workspace_bytes(C.byref(beam(batch=1 << 24, beams=1, vocab=1 << 30, n_out=128))) > 1 << 34
    assert time.monotonic() - t < 20


@pytest.mark.parametrize("parent", [2 * A, 2 * A + 508, 2 * A - 28])
@pytest.mark.parametrize("n", [1, 60])
def test_reorder_refuses_a_parent_in_a_destination(parent, n):
    """The parents are read by every block, also after others have written."""
    ts = (L.ReorderTensor * n)(*[tensor(src=(100 + 2 * i) * A, dst=(2 + 300 * i) * A) for i in range(n)])
    assert lib.llmoc_beam_reorder(ts, n, parent, 2, 4, 4, 0, None) == 1 and "parent" in L.last_error()
    assert lib.llmoc_beam_reorder(ts, n, 2 * A - 32, 2, 4, 4, 1 << 20, None) == 2  # beside it: only the device is missing
    assert lib.llmoc_beam_reorder(ts, n, ts[0].src, 2, 4, 4, 1 << 20, None) == 2


@pytest.mark.parametrize("kw", [dict(norm_out=A), dict(residual_out=2 * A + 126), dict(norm_out=3 * A - 510),
                                dict(residual_out=2 * A, ld_residual_out=72)])
def test_norm_refuses_outputs_over_weights(kw):
    assert lib.llmoc_norm_residual(C.byref(norm_desc()), C.byref(norm_io(**kw)), 4, 0, None) == 1, L.last_error()
    assert "overlaps a weight" in L.last_error()


def test_norm_takes_outputs_beside_weights():
    for kw in (dict(norm_out=A + 128), dict(residual_out=2 * A - 512)):
        assert lib.llmoc_norm_residual(C.byref(norm_desc()), C.byref(norm_io(**kw)), 4, 1 << 20, None) == 2


def test_linear_create_refuses_unaligned_scales():
    """On the device they are read as they lie; host buffers are copied first."""
    for kw in (dict(scales=2 * A + 1), dict(scheme=1, zeros=3 * A + 1)):
        h = C.c_void_p()
        assert lib.llmoc_int4_linear_create(views(**kw), 1, 1 << 20, 1, C.byref(h)) == 1 and "aligned" in L.last_error()
        assert lib.llmoc_int4_linear_create(views(**kw), 1, 1 << 20, 0, C.byref(h)) == 2
    assert lib.llmoc_int4_linear_create(views(zeros=3 * A + 1), 1, 1 << 20, 1, C.byref(h)) == 2  # not read
