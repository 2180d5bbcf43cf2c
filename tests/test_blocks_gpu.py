"""The training-block operators (lidarseg3d_amd/blocks.py) on the device: the cases of tests/block_cases.py, sizes of the training step, streams, captured steps,
the models' training forward on them."""
import pytest
import torch

from tests import block_cases as bc

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("case", bc.DROPOUT + [(2000, 192, bc.F32, 0.1, True), (1203, 1001, bc.BF16, 0.25, False), (70000, 8, bc.F16, 0.5, False)], ids=str)
def test_dropout(case):
    bc.run_dropout(case, DEV)


@pytest.mark.parametrize("case", bc.RESIDUAL_NORM + [
    (20011, 96, bc.F32, bc.F32, "layer", None, None, 1.0, 0.1, False),
    (1030, 2048, bc.BF16, bc.F32, "rms", "rms", "channel", 0.5, 0.0, True),
    (603, 771, bc.F16, bc.F16, "layer", None, "full", 1.25, 0.2, True),
    (5000, 64, bc.BF16, bc.BF16, "layer", "layer", "channel", 1.0, 0.1, True)], ids=str)
def test_residual_norm(case):
    bc.run_residual_norm(case, DEV)


@pytest.mark.parametrize("index", [torch.int32, torch.int64], ids=["i32", "i64"])
@pytest.mark.parametrize("case", bc.EMBEDDING + [
    (32, 64, bc.F32, (40000,), False, False, 1.0, "uniform"),
    (5000000, 2, bc.F32, (20000,), False, False, 1.0, "uniform"),
    (30000, 16, bc.BF16, (300000,), False, False, 1.0, "uniform"),
    (3, 64, bc.BF16, (30011,), False, False, 1.0, "few"),
    (20000, 48, bc.F32, (9000, 8), True, True, 1.0, "holes"),
    (2, 1024, bc.F16, (5003,), False, False, 1.0, "one"),
    (5000, 1024, bc.BF16, (4096,), False, False, 32.0, "uniform")], ids=str)
def test_embedding(case, index):
    bc.run_embedding(case, DEV, index=index)


def test_shapes_strides_and_absent_parts():
    bc.run_strides_and_absent_parts(DEV)


def test_partial_gradients_and_shared_inputs():
    bc.run_partial_gradients(DEV)


def test_masked_rows_and_values():
    bc.run_masked_rows(DEV)


@pytest.mark.parametrize("rows,width,table", [(12, 24, 30), (700, 96, 64)])
def test_a_block_of_all_three_operators(rows, width, table):
    bc.run_block(DEV, rows, width, table)


@pytest.mark.parametrize("points,p", [(300, 0.0), (300, 0.1), (70000, 0.1)])
def test_decoder_training_forward(points, p, monkeypatch):
    bc.run_decoder(DEV, points, p, monkeypatch)


def test_reader_training_forward():
    bc.run_reader(DEV, 5000)


def test_camera_sampling():
    bc.run_camera_sampling(DEV, 6000)


def test_use_in_training():
    bc.run_use_in_training(DEV)


def test_dropout_rate_and_independence_of_calls():
    """2^22 draws at p = 0.1: the share that is dropped is within 6 standard deviations, and two calls agree in p^2 + (1 - p)^2 of the places"""
    from lidarseg3d_amd import blocks
    st = blocks.DropoutState(5, device=DEV)
    x = torch.ones(1 << 14, 256, device=DEV)
    a, b = blocks.dropout(x, 0.1, st) != 0, blocks.dropout(x, 0.1, st) != 0
    n = x.numel()
    p = 6554 / 65536
    for share, q in ((1 - float(a.float().mean(dtype=torch.float64)), p), (float((a == b).float().mean(dtype=torch.float64)), p * p + (1 - p) ** 2)):
        assert abs(share - q) <= 6 * (q * (1 - q) / n) ** 0.5
    st.advance()
    c = blocks.dropout(x, 0.1, st) != 0
    assert not torch.equal(a, c) and st.calls == 1


def test_work_runs_on_the_current_stream():
    """inputs made and outputs used on a side stream, with the default stream busy"""
    from lidarseg3d_amd import blocks
    side = torch.cuda.Stream()
    st = blocks.DropoutState(7, device=DEV)
    x0 = torch.randn(4096, 256, device=DEV)
    tab0, ix = torch.randn(500, 256, device=DEV), torch.randint(0, 500, (4096,), device=DEV)

    def work():
        x, tab = x0.clone().requires_grad_(), tab0.clone().requires_grad_()
        y = blocks.residual_norm(blocks.dropout(x, 0.2, st.tensor, call=0), blocks.embedding(tab, ix), norm=blocks.Norm("layer"), p=0.1, state=st.tensor, call=1)
        return [y.detach()] + list(torch.autograd.grad(y, [x, tab], [x0]))
    want = [t.clone() for t in work()]
    side.wait_stream(torch.cuda.current_stream())
    busy = torch.randn(4096, 4096, device=DEV)
    for _ in range(10):
        busy = busy @ busy * 1e-2
    with torch.cuda.stream(side):
        got = work()
    torch.cuda.current_stream().wait_stream(side)
    for g, w in zip(got, want):
        assert torch.equal(g, w)


def test_captured_training_steps_draw_anew_and_equal_eager_steps():
    """two graphs of one training step each (forward, backward, update, advance), replayed in turn with eager work between, against the eager steps"""
    P = bc.block_parameters(torch.Generator().manual_seed(3), 96, 200, DEV)
    from lidarseg3d_amd import blocks
    gen = torch.Generator().manual_seed(4)
    batches = [(torch.randint(0, 200, (512,), generator=gen).to(DEV), torch.randn(512, 96, generator=gen).to(DEV)) for _ in range(6)]
    start = {k: v.detach().clone() for k, v in P.items()}

    def step(W, state, tokens, target, y_out):
        y, s = bc.block_forward(W, tokens, state, 0.2)
        grads = torch.autograd.grad([y, s], list(W.values()), [target, target])
        with torch.no_grad():
            y_out.copy_(y)
            for w, g in zip(W.values(), grads):
                w.sub_(g, alpha=1e-3)
        state.advance()

    def fresh():
        return {k: v.clone().requires_grad_() for k, v in start.items()}, blocks.DropoutState(11, device=DEV)
    W, state = fresh()
    out, want = torch.empty(512, 96, device=DEV), []
    for tokens, target in batches:
        step(W, state, tokens, target, out)
        want.append(out.clone())
    final = {k: v.detach().clone() for k, v in W.items()}
    del W
    W, state = fresh()
    side = torch.cuda.Stream()
    ins = [(batches[0][0].clone(), batches[0][1].clone(), torch.empty(512, 96, device=DEV)) for _ in range(2)]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # warm-up on throw-away weights
        T, ts = fresh()
        step(T, ts, *ins[0])
        del T
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for tokens, target, y in ins:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(W, state, tokens, target, y)
        graphs.append(g)
    for i, (tokens, target) in enumerate(batches):
        ins[i % 2][0].copy_(tokens)
        ins[i % 2][1].copy_(target)
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        assert torch.equal(ins[i % 2][2], want[i]), "replay %d" % i
        blocks.residual_norm(target, target, norm=blocks.Norm("rms"))  # the program's own work between replays
    for k in final:
        assert torch.equal(W[k].detach(), final[k]), k


def test_large_table_and_offsets_beyond_32_bits():
    """a table of more than 2^31 elements: the last rows are found and their gradient lands there; a dropout over more than 2^31 elements
    draws by row and column"""
    from lidarseg3d_amd import blocks
    rows, c = 1 << 19, 4104  # 2.15 G elements of bf16
    table = torch.zeros(rows, c, dtype=torch.bfloat16, device=DEV)
    table[-3:] = torch.randn(3, c, device=DEV).bfloat16()
    ix = torch.tensor([rows - 1, 0, rows - 3, rows - 1], device=DEV)
    table.requires_grad_()
    y = blocks.embedding(table, ix)
    assert torch.equal(y, table.detach()[ix])
    g = torch.randn(4, c, device=DEV).bfloat16()
    (dt,) = torch.autograd.grad(y, [table], [g])
    assert torch.equal(dt[rows - 1], (g[0].float() + g[3].float()).bfloat16()) and torch.equal(dt[rows - 3], g[2]) and torch.equal(dt[0], g[1])
    assert bool((dt[1:rows - 3] == 0).all()) and bool((dt[rows - 2] == 0).all())
    del dt, y
    st = blocks.DropoutState(9, device=DEV)
    z = blocks.dropout(table.detach().fill_(1.0), 0.5, st.tensor, call=0)
    keep, inv = bc.keep_mask(4, c, 0.5, 9, 0, 0)
    assert torch.equal(z[:4].cpu().float(), keep.float() * inv)
    big = z[rows - 64:].clone()
    del z
    s, t = blocks.residual_norm(table.detach(), norm=blocks.Norm("rms"), p=0.5, state=st.tensor, call=0, return_sum=True)[::-1]
    assert torch.equal(s[rows - 64:], big)


def test_large_passes_equal_their_parts():
    """passes of more than 256 MB take other accesses (non-temporal, more workgroups): bit for bit what their parts give, row by row"""
    from lidarseg3d_amd import blocks
    gen = torch.Generator(device=DEV).manual_seed(1)
    for n, c, T, kind in ((120001, 256, torch.float32, "layer"), (30001, 2050, torch.bfloat16, "rms"), (8193, 8191, torch.float16, "layer")):
        x, r, dy = (torch.randn(n, c, generator=gen, device=DEV).to(T) for _ in range(3))
        w = torch.randn(c, generator=gen, device=DEV, requires_grad=True)
        parts = [slice(a, min(a + n // 5, n)) for a in range(0, n, n // 5)]

        def run(sl, gate):
            xs, rs = x[sl].detach().requires_grad_(), r[sl].detach().requires_grad_()
            out = blocks.residual_norm(xs, rs, norm=blocks.Norm(kind, w), norm_in=blocks.Norm("rms", w) if gate else None, gate=w if gate else None, alpha=0.5, return_sum=True)
            return [t.detach() for t in out] + list(torch.autograd.grad(out, [xs, rs, w], [dy[sl], dy[sl]]))
        for gate in (False, True):
            whole, pieces = run(slice(0, n), gate), [run(sl, gate) for sl in parts]
            for i in range(4):
                assert torch.equal(whole[i], torch.cat([p[i] for p in pieces])), (n, c, T, gate, i)
            if not gate:  # dw = sum dy shat, here in float64 from the sum's values; terms added in f32, a thread's share of at most ceil(n / 512) + 64 in sequence
                s = whole[1].double()
                d = s - (s.mean(1, keepdim=True) if kind == "layer" else 0.0)
                terms = dy.double() * d / (d.square().mean(1, keepdim=True) + 1e-5).sqrt()
                # shat itself: K32 of the largest (|alpha r| + |x|) / std of a row, and the sum's rounding to its type
                off = (dy.double().abs() * (bc.K32 * 8 + bc.unit(T) * s.abs().amax(1, keepdim=True))).sum(0)
                assert bool(((whole[4].double() - terms.sum(0)).abs() <= (n / 512 + 64) * 2.0 ** -24 * terms.abs().sum(0) + off).all())
            del whole, pieces
        st = blocks.DropoutState(3, device=DEV)
        big = torch.cat([x, r, dy]) if T != torch.float32 else torch.cat([x, r])
        z = blocks.dropout(big, 0.3, st.tensor, call=5, relu=True)
        keep, inv = bc.keep_mask(64, c, 0.3, 3, 0, 5)
        want = torch.where(keep.to(DEV), torch.relu(big[:64].float()) * float(torch.tensor(inv, dtype=torch.float32)), torch.zeros((), device=DEV)).to(T)
        assert torch.equal(z[:64], want)
        assert torch.equal(z[:9000], blocks.dropout(big[:9000], 0.3, st.tensor, call=5, relu=True))
        del big, z


@pytest.mark.parametrize("reentrant", [False, True])
def test_activation_checkpointing(reentrant):
    bc.run_checkpointing(DEV, reentrant)


def test_accumulated_gradients():
    bc.run_accumulated_gradients(DEV)


def test_weight_gradient_of_no_columns():
    bc.run_weight_gradient_of_no_columns(DEV)


def test_forward_mode_is_refused():
    bc.run_forward_mode(DEV)


def test_tracers_and_wrapped_tensors_are_refused():
    bc.run_tracers_and_wrapped_tensors(DEV)


def test_converted_dropouts():
    bc.run_converted_dropouts(DEV)


def test_differentiated_evaluation():
    bc.run_differentiated_evaluation(DEV, 700)


def test_dropped_rows_beside_infinities():
    bc.run_dropped_rows_beside_infinities(DEV)


def test_rows_near_the_largest_value():
    bc.run_rows_near_the_largest_value(DEV)


def test_rows_of_equal_values():
    bc.run_rows_of_equal_values(DEV)


def test_single_value_gates():
    bc.run_single_value_gates(DEV)


def test_one_element_with_a_gate():
    bc.run_one_element_with_a_gate(DEV)


def test_camera_sampling_types():
    bc.run_camera_sampling_types(DEV)


def test_negated_views():
    bc.run_negated_views(DEV)


@pytest.mark.parametrize("index", [torch.int32, torch.int64], ids=["i32", "i64"])
@pytest.mark.parametrize("case", bc.EXACT_LOOKUP + bc.EXACT_LOOKUP_LARGE, ids=str)
def test_exact_lookup(case, index):
    bc.run_exact_lookup(case, DEV, index=index)


def test_exact_lookup_of_random_sizes():
    import random
    rng = random.Random(6)
    for i in range(60):
        bc.run_exact_lookup(bc.random_exact_lookup(rng, 20000000), DEV, seed=i, index=rng.choice([torch.int32, torch.int64]))


def test_inputs_changed_before_the_backward_pass():
    bc.run_inputs_changed_before_the_backward_pass(DEV)
