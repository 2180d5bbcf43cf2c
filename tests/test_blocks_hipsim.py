"""The training-block operators (lidarseg3d_amd/blocks.py) without a GPU: the kernels compiled for the host against tests/hipsim, driven through the
package's own entry points and checked against 64-bit references (tests/block_cases.py); the refusals."""
import os
import sys

import pytest
import torch

from lidarseg3d_amd import _lib, blocks, ops
from tests import block_cases as bc

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module", autouse=True)
def sim_library():
    sys.path.insert(0, os.path.join(HERE, "hipsim"))
    import build_sim
    from lidarseg3d_amd import build
    build.build_host()  # (only where it is missing or older than its source)
    _lib.use_library_for_testing(build_sim.build())
    ops.set_sim(True)
    yield
    ops.set_sim(False)
    _lib.use_library_for_testing(None)


def test_generator_against_the_published_known_answers():
    """the three known answers the authors of Philox publish with it, for the oracle; then every 16-bit draw of the kernel: p = t / 65536 moves the
    threshold, an element is kept exactly while its draw is not below it"""
    F = 0xFFFFFFFF
    assert bc.philox_words(0, 0, 0, 0, 0, 0) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    assert bc.philox_words(F, F, F, F, F, F) == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]
    assert bc.philox_words(0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344, 0xa4093822, 0x299f31d0) == [0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1]
    w = bc.philox_words(1, 2, 3, 4, 5, 6)  # group 1, row 2, call 3, step 4, seed 6 << 32 | 5
    draws = [h for x in w for h in (x & 0xFFFF, x >> 16)]
    state = torch.tensor([6 << 32 | 5, 4], dtype=torch.int64)
    x = torch.ones(3, 16)
    for j, d in enumerate(draws):
        assert float(blocks.dropout(x, d / 65536.0, state, call=3)[2, 8 + j]) != 0.0
        assert float(blocks.dropout(x, (d + 1) / 65536.0, state, call=3)[2, 8 + j]) == 0.0


@pytest.mark.parametrize("case", bc.DROPOUT, ids=str)
def test_dropout(case):
    bc.run_dropout(case, "cpu")


@pytest.mark.parametrize("case", bc.RESIDUAL_NORM, ids=str)
def test_residual_norm(case):
    bc.run_residual_norm(case, "cpu")


@pytest.mark.parametrize("index", [torch.int32, torch.int64], ids=["i32", "i64"])
@pytest.mark.parametrize("case", bc.EMBEDDING, ids=str)
def test_embedding(case, index):
    bc.run_embedding(case, "cpu", index=index)


@pytest.mark.parametrize("device", ["cpu"])
def test_shapes_strides_and_absent_parts(device):
    bc.run_strides_and_absent_parts(device)


def test_a_block_of_all_three_operators(device="cpu"):
    bc.run_block(device, rows=12, width=24, table=30)


def test_partial_gradients_and_shared_inputs():
    bc.run_partial_gradients("cpu")


def test_masked_rows_and_values():
    bc.run_masked_rows("cpu")


@pytest.mark.parametrize("p", [0.0, 0.1])
def test_decoder_training_forward(p, monkeypatch):
    bc.run_decoder("cpu", 23, p, monkeypatch)


def test_reader_training_forward():
    bc.run_reader("cpu", 11)


def test_camera_sampling():
    bc.run_camera_sampling("cpu", 60)


def test_use_in_training():
    bc.run_use_in_training("cpu")
    with pytest.raises(TypeError, match="DropoutState"):
        blocks.use_in_training(torch.nn.Linear(2, 2), torch.zeros(2, dtype=torch.int64))


def test_refusals():
    x, st = torch.randn(4, 8), blocks.DropoutState(1, device="cpu")
    N = blocks.Norm("layer", torch.ones(8), torch.zeros(8))
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError, match="probability"):
            blocks.dropout(x, p, st)
    with pytest.raises(ValueError, match="DropoutState"):
        blocks.dropout(x, 0.5, None)
    with pytest.raises(ValueError, match="DropoutState"):
        blocks.dropout(x, 0.5, torch.zeros(2))
    with pytest.raises(ValueError, match="call"):
        blocks.dropout(x, 0.5, st.tensor)
    with pytest.raises(ValueError, match="call"):
        blocks.dropout(x, 0.5, st.tensor, call=1 << 32)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        blocks.dropout(x.double(), 0.5, st)
    with pytest.raises(ValueError, match="kind"):
        blocks.Norm("batch")
    with pytest.raises(ValueError, match="eps"):
        blocks.Norm("rms", eps=-1.0)
    with pytest.raises(ValueError, match="last dimension"):
        blocks.Norm.of(torch.nn.LayerNorm([4, 8]))
    with pytest.raises(ValueError, match="eps"):
        blocks.Norm.of(torch.nn.RMSNorm(8))
    with pytest.raises(TypeError, match="nn.LayerNorm"):
        blocks.Norm.of(torch.nn.BatchNorm1d(8)) if hasattr(torch.nn.BatchNorm1d(8), "normalized_shape") else blocks.Norm.of(type("M", (), {"normalized_shape": (8,)})())
    with pytest.raises(ValueError, match="residual"):
        blocks.residual_norm(x, x[:3], norm=N)
    with pytest.raises(TypeError, match="residual"):
        blocks.residual_norm(x, x.bfloat16(), norm=N)
    with pytest.raises(ValueError, match="gate"):
        blocks.residual_norm(x, x, norm=N, gate=torch.ones(7))
    with pytest.raises(TypeError, match="gate"):
        blocks.residual_norm(x, x, norm=N, gate=x.bfloat16())
    with pytest.raises(TypeError, match="Norm"):
        blocks.residual_norm(x, x, norm=torch.nn.LayerNorm(8))
    with pytest.raises(ValueError, match="weight"):
        blocks.residual_norm(x, x, norm=blocks.Norm("rms", torch.ones(7)))
    with pytest.raises(ValueError, match="8192"):
        blocks.residual_norm(torch.randn(1, 8193))
    t = torch.randn(5, 8)
    with pytest.raises(TypeError, match="indices"):
        blocks.embedding(t, torch.zeros(3))
    with pytest.raises(ValueError, match="table"):
        blocks.embedding(t[0], torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="match"):
        blocks.embedding(t, torch.zeros(3, 2, dtype=torch.int64), weight=torch.ones(3))
    with pytest.raises(TypeError, match="weights"):
        blocks.embedding(t, torch.zeros(3, 2, dtype=torch.int64), weight=torch.ones(3, 2).double())
    with pytest.raises(ValueError, match="no indices"):
        blocks.embedding(t, torch.zeros(3, 0, dtype=torch.int64), bag=True)
    with pytest.raises(ValueError, match="padding_idx"):
        blocks.embedding(t, torch.zeros(3, dtype=torch.int64), padding_idx=5)
    # drawn after a step: the backward pass would make another mask
    x.requires_grad_()
    y = blocks.dropout(x, 0.5, st)
    st.advance()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    # second derivatives are refused, not answered as if the first were constant
    for y, leaf in ((blocks.dropout(x, 0.5, st), x), (blocks.residual_norm(x, norm=N), x), (blocks.embedding(x, torch.zeros(3, dtype=torch.int64)), x)):
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(y.sum(), [leaf], create_graph=True)
    ops.set_sim(False)
    try:
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            blocks.dropout(x, 0.5, st)
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            blocks.residual_norm(x, x, norm=N)
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            blocks.embedding(t, torch.zeros(3, dtype=torch.int64))
    finally:
        ops.set_sim(True)


def test_argument_errors_of_the_c_entry_points():
    """every call that the kernels could not run within their buffers is answered with a code before anything is launched"""
    import ctypes
    L, ll, f = _lib.load(), ctypes.c_longlong, ctypes.c_float
    ARG, UNS, WS = -1, -3, -4
    x, y, st = torch.zeros(64), torch.zeros(64), torch.zeros(2, dtype=torch.int64)
    P = lambda t, off=0: ctypes.c_void_p(t.data_ptr() + off)
    u = ctypes.c_uint32(0)
    ok = lambda **k: L.ls3d_dropout_forward(k.get("x", P(x)), ll(k.get("ld", 8)), ll(k.get("rows", 8)), ll(8), k.get("dt", 0), f(k.get("p", 0.5)), k.get("st", P(st)), u,
                                            0, k.get("y", P(y)), None, None)
    assert ok() == 0 and ok(rows=0, x=None, y=None, st=None) == 0
    for bad in (dict(ld=7), dict(rows=-1), dict(dt=3), dict(p=1.5), dict(p=float("nan")), dict(st=None), dict(st=P(st, 4)), dict(x=None), dict(y=None), dict(x=P(x, 2))):
        assert ok(**bad) == ARG, bad
    assert L.ls3d_dropout_backward(P(x), ll(8), None, ll(8), ll(8), 0, f(0.5), P(st), u, 1, P(y), None) == ARG  # relu: the bits are needed
    d = _lib.ResidualNorm()
    d.out.kind, d.alpha = 1, 1.0
    stats, ws = torch.zeros(8, 4), torch.zeros(1 << 16, dtype=torch.uint8)
    fwd = lambda **k: L.ls3d_residual_norm_forward(k.get("x", P(x)), ll(k.get("ld", 8)), k.get("r", P(x)), ll(k.get("rld", 8)), k.get("n", 8), k.get("c", 8), ctypes.byref(d),
                                                   k.get("y", P(y)), None, k.get("stats", P(stats)), None)
    assert fwd() == 0 and fwd(n=0, x=None, r=None, y=None) == 0 and fwd(c=8193, ld=8193) == UNS
    for bad in (dict(ld=7), dict(rld=7), dict(n=-1), dict(x=None), dict(y=None), dict(stats=P(stats, 4)), dict(r=P(x, 2))):
        assert fwd(**bad) == ARG, bad
    for field, value, code in (("dtype", 3, ARG), ("gate_kind", 3, ARG), ("gate_kind", 1, ARG), ("p", 0.5, ARG), ("p", -1.0, ARG), ("dtype", 1, 0), ("stream_dtype", 1, UNS)):
        keep = getattr(d, field)
        setattr(d, field, value)
        assert fwd() == code, (field, value)
        setattr(d, field, keep)
    d.out.kind = 3
    assert fwd() == ARG
    d.out.kind = 1
    g, dw = torch.zeros(64), torch.zeros(8)
    bwd = lambda **k: L.ls3d_residual_norm_backward(P(x), ll(8), P(x), ll(8), k.get("n", 8), 8, ctypes.byref(d), k.get("stats", P(stats)), k.get("dy", P(x)), ll(k.get("yld", 8)),
                                                    None, ll(0), k.get("dx", P(g)), None, k.get("dg"), k.get("dwi"), None, P(dw), None, k.get("ws", P(ws)),
                                                    ctypes.c_size_t(k.get("wsb", ws.numel())), None)
    assert bwd() == 0 and bwd(n=0) == 0
    for bad, code in ((dict(stats=None), ARG), (dict(dy=None), ARG), (dict(yld=7), ARG), (dict(ws=None), ARG), (dict(wsb=16), WS), (dict(dwi=P(dw)), ARG), (dict(dg=P(g)), ARG),
                      (dict(dx=P(g, 2)), ARG)):
        assert bwd(**bad) == code, bad
    idx, big = torch.zeros(8, dtype=torch.int64), torch.zeros(1 << 20, dtype=torch.uint8)
    emb = lambda **k: L.ls3d_embedding_forward(k.get("t", P(x)), ll(k.get("ld", 8)), ll(k.get("rows", 8)), 8, k.get("dt", 0), k.get("ix", P(idx)), k.get("it", 1), k.get("n", 8),
                                               k.get("k", 1), None, f(1.0), k.get("y", P(y)), None)
    assert emb() == 0 and emb(n=0) == 0 and emb(rows=0, t=None) == 0
    for bad, code in ((dict(t=None), ARG), (dict(ld=7), ARG), (dict(rows=-1), ARG), (dict(dt=5), ARG), (dict(ix=None), ARG), (dict(ix=P(idx, 4)), ARG), (dict(it=2), ARG),
                      (dict(k=0), ARG), (dict(n=1 << 29, k=2), UNS), (dict(y=None), ARG)):
        assert emb(**bad) == code, bad
    eb = lambda **k: L.ls3d_embedding_backward(k.get("t"), ll(8), ll(8), 8, 0, P(idx), 1, 8, 1, None, f(1.0), ll(-1), k.get("do", P(x)), ll(k.get("old", 8)), P(y), k.get("dw"),
                                               k.get("ws", P(big)), ctypes.c_size_t(k.get("wsb", big.numel())), None)
    assert eb() == 0
    for bad, code in ((dict(do=None), ARG), (dict(old=7), ARG), (dict(ws=None), ARG), (dict(wsb=64), WS), (dict(ws=P(big, 4)), ARG), (dict(dw=P(dw)), ARG)):
        assert eb(**bad) == code, bad


@pytest.mark.parametrize("reentrant", [False, True])
def test_activation_checkpointing(reentrant):
    """a repeated forward pass draws the masks of the first with `call` given, and is refused where it would count on"""
    bc.run_checkpointing("cpu", reentrant)


def test_accumulated_gradients():
    bc.run_accumulated_gradients("cpu")


def test_weight_gradient_of_no_columns():
    bc.run_weight_gradient_of_no_columns("cpu")


def test_c_entry_of_a_weight_gradient_of_no_columns():
    """the indices are checked there too: they are read"""
    import ctypes
    L, ll, dw, idx = _lib.load(), ctypes.c_longlong, torch.full((8,), 7.0), torch.zeros(9, dtype=torch.int64)
    call = lambda ix: L.ls3d_embedding_backward(None, ll(0), ll(5), 0, 0, ix, 1, 8, 1, None, ctypes.c_float(1.0), ll(-1), None, ll(0), None, ctypes.c_void_p(dw.data_ptr()),
                                                None, ctypes.c_size_t(0), None)
    assert call(None) == -1 and call(ctypes.c_void_p(idx.data_ptr() + 4)) == -1 and bool((dw == 7).all())
    assert call(ctypes.c_void_p(idx.data_ptr())) == 0 and bool((dw == 0).all())


def test_forward_mode_is_refused():
    bc.run_forward_mode("cpu")


def test_tracers_and_wrapped_tensors_are_refused():
    bc.run_tracers_and_wrapped_tensors("cpu")


def test_converted_dropouts():
    bc.run_converted_dropouts("cpu")


def test_differentiated_evaluation():
    bc.run_differentiated_evaluation("cpu", 23)


def test_dropped_rows_beside_infinities():
    bc.run_dropped_rows_beside_infinities("cpu")


def test_rows_near_the_largest_value():
    bc.run_rows_near_the_largest_value("cpu")


def test_rows_of_equal_values():
    bc.run_rows_of_equal_values("cpu")


def test_single_value_gates():
    bc.run_single_value_gates("cpu")


def test_one_element_with_a_gate():
    bc.run_one_element_with_a_gate("cpu")


def test_learned_numbers_are_refused():
    """alpha and scale are numbers: as learned tensors they would be read and never get a gradient; tensors that want none are read"""
    x, table, ix = torch.ones(2, 4), torch.ones(3, 4), torch.tensor([0, 2])
    for learned in (torch.tensor(2.0, requires_grad=True), torch.nn.Parameter(torch.ones(1))):
        with pytest.raises(TypeError, match="alpha is a number"):
            blocks.residual_norm(x, x, alpha=learned)
        with pytest.raises(TypeError, match="scale is a number"):
            blocks.embedding(table, ix, scale=learned)
    assert bool((blocks.residual_norm(x, x, alpha=torch.tensor(2.0)) == 3).all()) and bool((blocks.embedding(table, ix, scale=torch.tensor(2.0)) == 2).all())


def test_camera_sampling_types():
    bc.run_camera_sampling_types("cpu")


def test_negated_views():
    bc.run_negated_views("cpu")


@pytest.mark.parametrize("case", bc.EXACT_LOOKUP + [(700, 64, bc.F32, (300000,), False, 1.0, "text")], ids=str)
def test_exact_lookup(case):
    bc.run_exact_lookup(case, "cpu")


def test_exact_lookup_of_random_sizes():
    import random
    rng = random.Random(5)
    for i in range(60):
        bc.run_exact_lookup(bc.random_exact_lookup(rng, 60000), "cpu", seed=i, index=rng.choice([torch.int32, torch.int64]))


def test_inputs_changed_before_the_backward_pass():
    bc.run_inputs_changed_before_the_backward_pass("cpu")
