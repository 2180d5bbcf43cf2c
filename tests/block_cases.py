"""Shared by test_blocks_hipsim.py (kernel logic on the host) and test_blocks_gpu.py: the training-block operators (lidarseg3d_amd/blocks.py) against
plain implementations in 64 bits, with error bounds that follow from the arithmetic.

A result is off by its own rounding, half a step of its type (u = eps / 2 of the value), and by what 32-bit arithmetic does before: each 32-bit operation
is off by 2^-24 of its result, a sum of up to 8192 values is 32 additions a lane and a tree of 8 (40 steps), and at most three such sums are nested.
(40 * 3 + a handful of products) < 128, so the bound is u |ref| + 128 * 2^-24 * scale, `scale` being the largest magnitude that enters the
subtractions on the way; it is computed beside the reference.  Column sums over n rows add at most ceil(n / blocks) + 64 terms in sequence."""
import numpy as np
import torch

K32 = 128 * 2.0 ** -24


def philox_words(c0, c1, c2, c3, k0, k1):
    """Philox4x32, 10 rounds, on Python integers: the definition, one counter at a time"""
    x, k = [c0, c1, c2, c3], [k0, k1]
    for _ in range(10):
        a, b = x[0] * 0xD2511F53, x[2] * 0xCD9E8D57
        x = [(b >> 32) ^ x[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ x[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return x


def keep_mask(rows, c, p, seed, step, call):
    """[rows, c] truth values, and the factor of what is kept (numpy, vectorised over the counters)"""
    u = np.uint64
    g = (c + 7) // 8
    x = [np.tile(np.arange(g, dtype=u), (rows, 1)), np.tile(np.arange(rows, dtype=u)[:, None], (1, g)), np.full((rows, g), call, u),
         np.full((rows, g), step % 2 ** 32, u)]
    k0, k1 = seed % 2 ** 32, (seed >> 32) % 2 ** 32
    for _ in range(10):
        a, b = x[0] * u(0xD2511F53), x[2] * u(0xCD9E8D57)
        x = [(b >> u(32)) ^ x[1] ^ u(k0), b & u(0xFFFFFFFF), (a >> u(32)) ^ x[3] ^ u(k1), a & u(0xFFFFFFFF)]
        k0, k1 = (k0 + 0x9E3779B9) % 2 ** 32, (k1 + 0xBB67AE85) % 2 ** 32
    draws = np.stack([(w >> u(s)) & u(0xFFFF) for w in x for s in (0, 16)], -1).reshape(rows, 8 * g)[:, :c]
    t = int(np.floor(65536 * float(np.float32(p)) + 0.5))
    return torch.from_numpy(np.ascontiguousarray(draws >= t)), (65536.0 / (65536 - t) if t < 65536 else 0.0)


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def check(got, ref, scale, what="", k=K32):
    """|got - ref| <= u |ref| + k * scale, element by element (scale broadcasts); half a smallest step besides, for values below the normal range"""
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    if ref.numel() == 0:
        return
    g = got.detach().cpu().double()
    assert torch.equal(torch.isnan(g), torch.isnan(ref)), what + ": NaN in other places"
    bound = unit(got.dtype) * ref.abs() + k * torch.as_tensor(scale, dtype=torch.float64) + torch.finfo(got.dtype).tiny * unit(got.dtype) * 2
    bad = (g - ref).abs() - bound
    bad = torch.where(torch.isnan(ref) | (g == ref), torch.full_like(bad, -1.0), bad)
    i = int(bad.argmax())
    assert float(bad.max()) <= 0, "%s: element %d is %.9g, reference %.9g, bound %.3g" % (what, i, float(g.reshape(-1)[i]), float(ref.reshape(-1)[i]),
                                                                                        float(bound.expand_as(ref).reshape(-1)[i]))


def _rmax(t):
    return t.abs().amax(1, keepdim=True)


def _norm(v, kind, w, b, eps):
    """-> value, hat, 1 / std in float64"""
    m = v.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(v[:, :1])
    r = 1.0 / ((v - m).square().mean(1, keepdim=True) + eps).sqrt()
    h = (v - m) * r
    y = h * w if w is not None else h
    return (y + b if b is not None else y), h, r


def _back(u, h, r, kind):
    g = u - h * (u * h).mean(1, keepdim=True)
    return r * (g - u.mean(1, keepdim=True)) if kind == "layer" else r * g


def residual_norm_reference(x, residual, norm, norm_in, gate, alpha, p, draw, dy, ds):
    """every output of residual_norm and every gradient by the formulas, in float64 on the host: name -> (reference, scale).  norm / norm_in:
    None or (kind, weight, bias, eps) of host tensors; draw: (seed, step, call); dy / ds: gradients or None"""
    D = lambda t: None if t is None else t.detach().cpu().double()
    x, residual, gate, dy, ds = D(x), D(residual), D(gate), D(dy), D(ds)
    w_in, b_in = (D(norm_in[1]), D(norm_in[2])) if norm_in else (None, None)
    w_out, b_out = (D(norm[1]), D(norm[2])) if norm else (None, None)
    mag = lambda t, other: other if t is None else float(t.abs().max())
    res = {}
    t, T = x, _rmax(x)
    if norm_in:
        t, xh, r_in = _norm(x, norm_in[0], w_in, b_in, norm_in[3])
        cond_in = T * r_in
        T = cond_in * (1 + _rmax(xh)) * mag(w_in, 1.0) + mag(b_in, 0.0)
    keep, inv = keep_mask(x.shape[0], x.shape[1], p, *draw) if p > 0 else (torch.ones(x.shape, dtype=torch.bool), 1.0)
    d = torch.where(keep, t * inv, torch.zeros(1, dtype=torch.float64))
    T = T * inv
    g = gate if gate is not None else torch.ones(1, dtype=torch.float64)
    gmax = float(g.abs().max())
    s = g * d + (alpha * residual if residual is not None else 0.0)
    Ss = gmax * T + (abs(alpha) * _rmax(residual) if residual is not None else 0.0)
    res["s"] = (s, Ss)
    G = torch.zeros_like(s)
    Gs = torch.zeros_like(Ss)
    if norm:
        y, sh, r_out = _norm(s, norm[0], w_out, b_out, norm[3])
        cond = Ss * r_out
        Hs = cond * (1 + _rmax(sh))
        res["y"] = (y, Hs * mag(w_out, 1.0) + mag(b_out, 0.0))
        if dy is not None:
            u = dy * w_out if w_out is not None else dy
            G = _back(u, sh, r_out, norm[0])
            Gs = r_out * _rmax(u) * (1 + _rmax(sh)) * (1 + Hs)
            res["w_out"], res["b_out"] = ((dy * sh).sum(0), (_rmax(dy) * Hs).sum()), (dy.sum(0), dy.abs().sum(0))
    if ds is not None:
        G, Gs = G + ds, Gs + _rmax(ds)
    if dy is None and ds is None:
        return res
    res["residual"] = (alpha * G, abs(alpha) * Gs)
    if gate is not None:
        res["gate"] = (G * d, Gs * T) if gate.dim() == 2 else ((G * d).sum(0), (Gs * T).sum())
    dt = torch.where(keep, g * G * inv, torch.zeros(1, dtype=torch.float64))
    Dt = gmax * Gs * inv
    if norm_in:
        res["w_in"], res["b_in"] = ((dt * xh).sum(0), (Dt * (1 + cond_in)).sum()), (dt.sum(0), Dt.sum())
        u = dt * w_in if w_in is not None else dt
        res["x"] = (_back(u, xh, r_in, norm_in[0]), r_in * Dt * mag(w_in, 1.0) * (1 + _rmax(xh)) * (1 + cond_in * (1 + _rmax(xh))))
    else:
        res["x"] = (dt, Dt)
    return res


def embedding_reference(table, idx, weight, scale, padding, dy, bag):
    """(out, scale), (dtable, scale), (dweight, scale) in float64, entry by entry in input order"""
    t, g = table.detach().cpu().double(), dy.detach().cpu().double()
    c, rows = t.shape[1], t.shape[0]
    ix = idx.cpu().long().reshape(-1, idx.shape[-1] if bag else 1)
    n, k = ix.shape
    w = weight.detach().cpu().double().reshape(n, k) if weight is not None else torch.ones(n, k, dtype=torch.float64)
    g = g.reshape(n, c)
    out, out_s = torch.zeros(n, c, dtype=torch.float64), torch.zeros(n, c, dtype=torch.float64)
    dt, dt_s = torch.zeros_like(t), torch.zeros_like(t)
    dw, dw_s = torch.zeros(n, k, dtype=torch.float64), torch.zeros(n, k, dtype=torch.float64)
    for j in range(k):
        hit = torch.nonzero((ix[:, j] >= 0) & (ix[:, j] < rows))[:, 0]
        v = ix[hit, j]
        term = scale * w[hit, j].unsqueeze(1) * t[v]
        out[hit] += term
        out_s[hit] += term.abs()
        dw[hit, j], dw_s[hit, j] = scale * (t[v] * g[hit]).sum(1), abs(scale) * (t[v] * g[hit]).abs().sum(1)
        if padding is not None:
            hit = hit[v != padding]
            v = ix[hit, j]
        term = scale * w[hit, j].unsqueeze(1) * g[hit]
        dt.index_add_(0, v, term)
        dt_s.index_add_(0, v, term.abs())
    return (out, out_s), (dt, dt_s), (dw, dw_s)


# ---------------------------------------------------------------------------------------------- sizes and forms
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16

# rows, c, x type, stream type, norm, norm_in, gate, alpha, p, return_sum: one token, one column, widths of every shape rule (4 / 16 / 64 / 256 lanes), odd and
# even, either side of each border, rows that leave lanes and workgroups idle
RESIDUAL_NORM = [
    (1, 1, F32, F32, "layer", None, None, 1.0, 0.0, False),
    (3, 7, F32, F32, "rms", "layer", "full", 1.5, 0.3, True),
    (70, 8, BF16, BF16, "layer", None, "channel", 1.0, 0.5, True),
    (66, 33, F16, F16, "layer", "rms", None, 0.5, 0.1, False),
    (131, 96, F32, F32, "layer", None, None, 1.0, 0.1, False),
    (13, 96, F32, F32, "layer", None, None, 1.0, 0.0, True),
    (14, 200, BF16, BF16, "rms", None, None, 1.0, 0.0, False),
    (9, 96, BF16, F32, None, "layer", "channel", 1.0, 0.25, True),
    (17, 128, F16, F32, "rms", "rms", "full", 1.0, 0.0, True),
    (20, 129, F32, F32, "rms", None, "channel", -1.0, 0.2, True),
    (18, 257, BF16, F32, "layer", "layer", None, 1.0, 0.1, True),
    (5, 512, F16, F16, "rms", None, "scalar", 2.0, 0.9, False),
    (6, 513, F32, F32, "layer", "rms", "channel", 1.0, 0.1, True),
    (4, 771, F16, F16, "layer", None, "full", 1.25, 0.2, True),
    (3, 1536, BF16, BF16, "rms", "rms", None, 1.0, 0.0, True),
    (5, 2047, BF16, F32, "layer", None, None, 1.0, 0.1, False),
    (3, 2049, F32, F32, "layer", "layer", "full", 1.0, 0.1, True),
    (1, 4096, BF16, BF16, "rms", None, None, 1.0, 0.0, True),
    (2, 6145, F16, F32, "rms", "layer", "channel", 0.5, 0.1, True),
    (2, 8192, BF16, BF16, "layer", None, None, 1.0, 0.4, False),
]

# rows, c, type, p, relu
DROPOUT = [(1, 1, F32, 0.5, False), (68, 96, F32, 0.1, False), (5, 7, BF16, 0.3, True), (33, 192, F32, 0.1, True), (11, 1001, BF16, 0.25, False), (3, 4099, F16, 0.9, True),
           (4, 64, F16, 1.0, False), (1, 5000, F32, 0.05, False), (7, 8, BF16, 1e-4, False)]

# table rows, c, type, index shape, bag, weights, scale, how the tokens fall
EMBEDDING = [
    (5, 1, F32, (1,), False, False, 1.0, "uniform"),
    (7, 9, BF16, (3, 5), False, False, 2.0, "uniform"),
    (40, 96, F32, (200,), False, False, 1.0, "uniform"),
    (3, 64, F32, (500,), False, False, 1.0, "few"),
    (1, 17, F16, (333,), False, False, 0.5, "few"),
    (1000, 33, F16, (257,), False, False, 1.0, "uniform"),
    (50, 48, F32, (60, 8), True, True, 1.0, "holes"),
    (30, 130, BF16, (40, 3), True, True, 4.0, "holes"),
    (30, 24, F32, (2, 9, 3), True, False, 1.0, "holes"),
    (70000, 5, F32, (90,), False, False, 1.0, "uniform"),
    (12, 1030, BF16, (70,), False, False, 32.0, "few"),
    (9, 64, F32, (1300,), False, False, 1.0, "one"),
    (2500, 3, F32, (5000,), False, False, 1.0, "uniform"),
    (150, 5, F32, (4000,), False, False, 1.0, "runs"),
    (64, 3, F32, (2000,), False, False, 1.0, "runs"),
    # more entries than one workgroup sorts: radix passes of one digit, of two, with entries that name no row
    (300, 2, F32, (16500,), False, False, 1.0, "uniform"),
    (9000, 3, F16, (17001,), False, False, 1.0, "uniform"),
    (70, 4, F32, (6000, 3), True, True, 1.0, "holes"),
]


def tensor(gen, *shape, dtype=F32, scale=1.0, shift=0.0, device="cpu"):
    return (torch.randn(*shape, generator=gen) * scale + shift).to(dtype).to(device)


def indices(gen, rows, shape, how, device, dtype=torch.int64):
    if how == "one":
        ix = torch.full(shape, rows - 1)
    elif how == "runs":  # rows named 1, 2, ... 70 times: they begin, end and fill up at every place of a tile
        ix = torch.repeat_interleave(torch.arange(rows), torch.arange(rows) % 70 + 1)[:shape[0]]
        ix = torch.cat([ix, torch.randint(0, rows, (shape[0] - ix.numel(),), generator=gen)])[torch.randperm(shape[0], generator=gen)]
    elif how == "few":
        ix = torch.randint(0, min(rows, 3), shape, generator=gen)
    else:
        ix = torch.randint(0, rows, shape, generator=gen)
    if how == "holes":  # rows that name nothing, and some beyond either end of the table
        ix = torch.where(torch.rand(shape, generator=gen) < 0.4, torch.full(shape, -1), ix)
        ix.reshape(-1)[0], ix.reshape(-1)[1] = rows, -7
        ix[1] = -1
    return ix.to(dtype).to(device)


def run_residual_norm(case, device, seed=0):
    """one case forward and backward through blocks.residual_norm, checked against the formulas"""
    from lidarseg3d_amd import blocks
    n, c, T, R, kind, kind_in, gate_kind, alpha, p, want_sum = case
    gen = torch.Generator().manual_seed(seed + n * 131 + c)
    mk = lambda *s, **kw: tensor(gen, *s, device=device, **kw).requires_grad_()
    x, res = mk(n, c, dtype=T), mk(n, c, dtype=R, scale=2.0)
    norm = (kind, mk(c, dtype=R, scale=0.1, shift=1.0), mk(c, dtype=T, scale=0.1) if kind == "layer" else None, 1e-5) if kind else None
    norm_in = (kind_in, mk(c, dtype=T, scale=0.1, shift=1.0), mk(c, scale=0.1) if kind_in == "layer" else None, 1e-6) if kind_in else None
    gate = {None: None, "full": lambda: mk(n, c, dtype=T), "channel": lambda: mk(c, dtype=R), "scalar": lambda: mk(1, dtype=F32)}[gate_kind]
    gate = gate() if gate else None
    state = blocks.DropoutState(0x123456789ABCDEF + seed, device=device, step=5)
    state.calls = 7
    mod = lambda m: blocks.Norm(m[0], m[1], m[2], m[3]) if m else None
    out = blocks.residual_norm(x, res, norm=mod(norm), norm_in=mod(norm_in), gate=gate, alpha=alpha, p=p, state=state, return_sum=want_sum)
    y, s = (out if want_sum else (out, None)) if kind else (None, out)
    dy = tensor(gen, n, c, dtype=T, device=device) if y is not None else None
    ds = tensor(gen, n, c, dtype=R, device=device) if s is not None else None
    leaves = dict(x=x, residual=res)
    for nm, tag in ((norm, "out"), (norm_in, "in")):
        if nm:
            leaves["w_" + tag] = nm[1]
            if nm[2] is not None:
                leaves["b_" + tag] = nm[2]
    if gate is not None:
        leaves["gate"] = gate
    grads = torch.autograd.grad([t for t in (y, s) if t is not None], list(leaves.values()), [t for t in (dy, ds) if t is not None])
    ref = residual_norm_reference(x, res, norm, norm_in, gate.detach().expand(c) if gate_kind == "scalar" else gate, alpha, p, (0x123456789ABCDEF + seed, 5, 7), dy, ds)
    if y is not None:
        check(y, *ref["y"], what="y")
    if s is not None:
        check(s, *ref["s"], what="s")
    for name, g in zip(leaves, grads):
        r, sc = ref[name]
        if name == "gate" and gate_kind == "scalar":  # autograd adds the c channel gradients up, each rounded to f32
            r, sc = r.sum().reshape(1), sc * c
        check(g, r, sc, what="d " + name)


def run_dropout(case, device, seed=0):
    from lidarseg3d_amd import blocks
    n, c, T, p, relu = case
    gen = torch.Generator().manual_seed(seed + n + c)
    x = tensor(gen, n, c, dtype=T, device=device)
    if x.numel() > 20:
        x.reshape(-1)[::9] = float("nan")  # behind the mask nothing of it is seen
        x.reshape(-1)[1::9] = float("inf")
    x.requires_grad_()
    dy = tensor(gen, n, c, dtype=T, device=device)
    state = blocks.DropoutState(-5 - seed, device=device, step=2 ** 32 + 3)
    y = blocks.dropout(x, p, state, call=9, relu=relu)
    (dx,) = torch.autograd.grad(y, [x], [dy])
    keep, inv = keep_mask(n, c, p, (-5 - seed) % 2 ** 64, 3, 9)
    zero = torch.zeros(1, dtype=torch.float64)
    xd = x.detach().cpu().double()
    want = torch.where(keep, (torch.relu(xd) if relu else xd) * inv, zero)
    got = y.detach().cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got) & torch.isinf(want), torch.isinf(want))
    fin = torch.isfinite(want)
    # one product in f32 by a factor that is itself rounded to f32, then the rounding to the type
    check(torch.where(fin.to(y.device), y.detach(), torch.zeros_like(y)), torch.where(fin, want, zero), torch.where(fin, want, zero).abs(), what="y")
    live = keep & ~(xd <= 0) if relu else keep
    ref = torch.where(live, dy.cpu().double() * inv, zero)
    check(dx, ref, ref.abs(), what="dx")


def run_embedding(case, device, seed=0, index=torch.int64):
    from lidarseg3d_amd import blocks
    rows, c, T, shape, bag, weights, scale, how = case
    gen = torch.Generator().manual_seed(seed + rows + c)
    table = tensor(gen, rows, c, dtype=T, device=device).requires_grad_()
    idx = indices(gen, rows, shape, how, device, index)
    weight = torch.rand(shape, generator=gen).to(device).requires_grad_() if weights else None
    padding = rows // 2 if how == "uniform" and rows > 20 else None
    y = blocks.embedding(table, idx, weight=weight, scale=scale, padding_idx=padding, bag=bag)
    assert y.shape == (*(shape[:-1] if bag else shape), c)
    dy = tensor(gen, *y.shape, dtype=T, device=device)
    grads = torch.autograd.grad(y, [table] + ([weight] if weights else []), [dy])
    out, dt, dw = embedding_reference(table, idx, weight, scale, padding, dy, bag)
    check(y.reshape(-1, c), *out, what="out")
    # a row's entries: <= `tile` in sequence, then a partial sum a tile
    check(grads[0], *dt, what="dtable", k=(np.prod(shape) + 16) * 2.0 ** -24)
    if weights:
        check(grads[1].reshape(dw[0].shape), *dw, what="dweight")
    again = torch.autograd.grad(blocks.embedding(table, idx, weight=weight, scale=scale, padding_idx=padding, bag=bag), [table], [dy])[0]
    assert torch.equal(again, grads[0])


def run_strides_and_absent_parts(device):
    """leading dimensions, column slices, transposed and expanded tensors, empty tensors; norms without weights, no residual, outputs that nothing uses"""
    from lidarseg3d_amd import blocks
    gen = torch.Generator().manual_seed(11)
    wide = tensor(gen, 6, 40, device=device)
    x = wide[:, 5:24]  # rows 40 apart that start anywhere
    res = tensor(gen, 19, 6, device=device).t()  # columns contiguous
    y, s = blocks.residual_norm(x, res, norm=blocks.Norm("layer"), return_sum=True)
    ref = residual_norm_reference(x, res, ("layer", None, None, 1e-5), None, None, 1.0, 0.0, None, None, None)
    check(y, *ref["y"], what="y of a slice")
    check(s, *ref["s"], what="s of a slice")
    x3 = tensor(gen, 2, 3, 19, device=device)
    y3 = blocks.residual_norm(x3, norm=blocks.Norm("rms"))
    ref = residual_norm_reference(x3.reshape(6, 19), None, ("rms", None, None, 1e-5), None, None, 1.0, 0.0, None, None, None)
    assert y3.shape == x3.shape
    check(y3.reshape(6, 19), *ref["y"], what="y of [2, 3, 19]")
    # a norm without parameters, its output unused: only the sum's gradient arrives; an expanded gradient (of .sum())
    x4, r4 = x3.clone().requires_grad_(), tensor(gen, 2, 3, 19, device=device).requires_grad_()
    w = torch.ones(19, device=device, requires_grad=True)
    y4, s4 = blocks.residual_norm(x4, r4, norm=blocks.Norm("layer", w), alpha=0.5, return_sum=True)
    dx, dr, dw = torch.autograd.grad(s4.sum(), [x4, r4, w])
    assert bool((dx == 1).all()) and bool((dr == 0.5).all()) and bool((dw == 0).all())
    dx, = torch.autograd.grad(blocks.residual_norm(x4, r4, norm=blocks.Norm("layer", w)).sum(), [x4])
    ref = residual_norm_reference(x4.reshape(6, 19), r4.reshape(6, 19), ("layer", w, None, 1e-5), None, None, 1.0, 0.0, None, torch.ones(6, 19), None)
    check(dx.reshape(6, 19), *ref["x"], what="dx of a summed norm")
    # no norm at all: the residual sum alone; nothing to differentiate; 1-D input
    z = blocks.residual_norm(x3, x3, alpha=2.0)
    check(z.reshape(6, 19), x3.cpu().double().reshape(6, 19) * 3, x3.cpu().double().reshape(6, 19).abs() * 3, what="plain sum")
    assert blocks.residual_norm(x3[0, 0], norm=blocks.Norm("rms")).shape == (19,)
    # empty tensors, both ways
    e = torch.zeros(0, 24, device=device, requires_grad=True)
    w24 = torch.ones(24, device=device, requires_grad=True)
    ye = blocks.residual_norm(e, e, norm=blocks.Norm("layer", w24))
    ge, gw = torch.autograd.grad(ye, [e, w24], [torch.zeros(0, 24, device=device)])
    assert ye.shape == (0, 24) and ge.shape == (0, 24) and bool((gw == 0).all())
    st = blocks.DropoutState(3, device=device)
    assert blocks.dropout(e, 0.5, st).shape == (0, 24)
    assert blocks.dropout(x3, 0.0, None) is x3 and bool((blocks.dropout(x3, 0.0, None, relu=True) == torch.relu(x3)).all())
    # dropout of a slice equals the slice's copy: the mask goes by row and column, not by address
    assert torch.equal(blocks.dropout(x, 0.4, st.tensor, call=1), blocks.dropout(x.contiguous(), 0.4, st.tensor, call=1))
    # tables and gradients with strides; an empty batch and a table nobody names
    tab = tensor(gen, 9, 40, device=device)[:, 3:20].requires_grad_()
    ix = torch.tensor([[0, 8], [3, 3]], device=device)
    out = blocks.embedding(tab, ix)
    assert torch.equal(out, tab[ix])
    g = tensor(gen, 2, 17, 2, device=device).transpose(1, 2)
    (dt,) = torch.autograd.grad(out, [tab], [g])
    want = torch.zeros(9, 17, dtype=torch.float64).index_add_(0, ix.cpu().reshape(-1), g.cpu().double().reshape(-1, 17))
    check(dt, want, want.abs(), what="dtable")
    t0 = torch.ones(4, 8, device=device, requires_grad=True)
    o0 = blocks.embedding(t0, torch.zeros(0, dtype=torch.int32, device=device))
    assert o0.shape == (0, 8) and bool((torch.autograd.grad(o0, [t0], [torch.zeros(0, 8, device=device)])[0] == 0).all())
    tz = torch.ones(0, 8, device=device, requires_grad=True)
    oz = blocks.embedding(tz, torch.tensor([0, 3, -1], device=device))
    assert oz.shape == (3, 8) and bool((oz == 0).all()) and torch.autograd.grad(oz.sum(), [tz])[0].shape == (0, 8)
    on = blocks.embedding(t0, torch.full((5,), -1, device=device))
    assert bool((on == 0).all()) and bool((torch.autograd.grad(on.sum(), [t0])[0] == 0).all())


def run_partial_gradients(device):
    """any subset of the inputs may want a gradient: each alone gives the bits it gives among all; one tensor as x and residual, as both norms' weight"""
    from lidarseg3d_amd import blocks
    gen = torch.Generator().manual_seed(21)
    base = dict(x=tensor(gen, 7, 40, device=device), residual=tensor(gen, 7, 40, device=device), gate=tensor(gen, 40, device=device), wi=tensor(gen, 40, device=device),
                bi=tensor(gen, 40, device=device), wo=tensor(gen, 40, device=device), bo=tensor(gen, 40, device=device))
    dy, ds = tensor(gen, 7, 40, device=device), tensor(gen, 7, 40, device=device)
    st = blocks.DropoutState(2, device=device)

    def run(names):
        t = {k: v.clone().requires_grad_(k in names) for k, v in base.items()}
        out = blocks.residual_norm(t["x"], t["residual"], norm=blocks.Norm("layer", t["wo"], t["bo"]), norm_in=blocks.Norm("layer", t["wi"], t["bi"]), gate=t["gate"], p=0.2,
                                   state=st.tensor, call=3, return_sum=True)
        return dict(zip(names, torch.autograd.grad(out, [t[k] for k in names], [dy, ds])))
    every = run(list(base))
    for name in base:
        assert torch.equal(run([name])[name], every[name]), name
    # x = residual: s = 2 x; the gradients of both places add up
    for p in (0.0, 0.3):
        x, w = base["x"].clone().requires_grad_(), base["wo"].clone().requires_grad_()
        y = blocks.residual_norm(x, x, norm=blocks.Norm("rms", w), norm_in=blocks.Norm("rms", w) if p else None, p=p, state=st.tensor, call=0)
        gx, gw = torch.autograd.grad(y, [x, w], [dy])
        ref = residual_norm_reference(x, x, ("rms", w, None, 1e-5), ("rms", w, None, 1e-5) if p else None, None, 1.0, p, (2, 0, 0), dy, None)
        check(gx, ref["x"][0] + ref["residual"][0], ref["x"][1] + ref["residual"][1], what="dx of both places")
        check(gw, ref["w_out"][0] + (ref["w_in"][0] if p else 0.0), ref["w_out"][1] + (ref["w_in"][1] if p else 0.0), what="dw of both places")
    # table and weights apart; rows that the same entry names twice
    tab, ix, wt = tensor(gen, 9, 16, device=device), torch.tensor([[1, 1, 4], [0, 4, 4]], device=device), torch.rand(2, 3, generator=gen).to(device)
    g = tensor(gen, 2, 16, device=device)
    both = [t.clone().requires_grad_() for t in (tab, wt)]
    dt, dw = torch.autograd.grad(blocks.embedding(both[0], ix, weight=both[1]), both, [g])
    t1, w1 = tab.clone().requires_grad_(), wt.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(blocks.embedding(t1, ix, weight=wt), [t1], [g])[0], dt)
    assert torch.equal(torch.autograd.grad(blocks.embedding(tab, ix, weight=w1), [w1], [g])[0], dw)
    ref = embedding_reference(tab, ix, wt, 1.0, None, g, True)
    check(dt, *ref[1], what="dtable of repeated rows")


def run_masked_rows(device):
    """everything dropped, rows of equal values, rows of the type's lowest value, infinities in dropped places"""
    from lidarseg3d_amd import blocks
    st = blocks.DropoutState(1, device=device)
    b = torch.arange(16.0, device=device)
    x = torch.full((3, 16), float("inf"), device=device).requires_grad_()
    y, s = blocks.residual_norm(x, torch.zeros(3, 16, device=device), norm=blocks.Norm("layer", None, b), p=1.0, state=st, return_sum=True)
    assert bool((s == 0).all()) and torch.equal(y, b.expand(3, 16))  # variance 0: the bias is left
    (dx,) = torch.autograd.grad([y, s], [x], [torch.ones_like(y), torch.ones_like(s)])
    assert bool((dx == 0).all())
    for T in (torch.float16, torch.bfloat16):  # their sum is beyond float32 for bf16
        lo = torch.full((2, 64), torch.finfo(T).min, dtype=T, device=device)
        y = blocks.residual_norm(lo, norm=blocks.Norm("layer"))
        assert bool((y == 0).all())  # all values alike: deviation 0
    r = blocks.residual_norm(torch.full((2, 64), 60000.0, dtype=torch.float16, device=device), norm=blocks.Norm("rms"))
    assert bool(((r.float() - 1).abs() <= 2.0 ** -11).all())
    # a NaN stays in its row
    z = torch.ones(3, 16, device=device)
    z[1, 2] = float("nan")
    y = blocks.residual_norm(z, norm=blocks.Norm("rms"))
    assert bool(torch.isnan(y[1]).all()) and not bool(torch.isnan(y[0]).any()) and not bool(torch.isnan(y[2]).any())
    # p = 1 of a bare dropout; relu keeps NaN like torch.relu
    assert bool((blocks.dropout(x, 1.0, st) == 0).all())
    # NaN in a table row nobody names, in a weight of an index that names none
    t = torch.ones(3, 4, device=device)
    t[1] = float("nan")
    w = torch.tensor([[1.0, float("nan")]], device=device)
    assert bool((blocks.embedding(t, torch.tensor([[0, -1]], device=device), weight=w) == 1).all())


def block_parameters(gen, width, table, device, dtype=torch.float32):
    mk = lambda *s, **k: tensor(gen, *s, dtype=dtype, device=device, **k).requires_grad_()
    return dict(table=mk(table, width), gate=mk(width, scale=0.5, shift=0.5), w1=mk(2 * width, width, scale=width ** -0.5), w2=mk(width, 2 * width, scale=(2 * width) ** -0.5),
                n1=mk(width, scale=0.1, shift=1.0), n2=mk(width, scale=0.1, shift=1.0), b2=mk(width, scale=0.1))


def block_forward(P, tokens, state, p):
    """embedding -> RMS norm before the block -> linear, dropout(relu), linear -> norm after it, gate, scaled residual, LayerNorm"""
    from lidarseg3d_amd import blocks
    F = torch.nn.functional
    h = blocks.embedding(P["table"], tokens, scale=2.0)
    y = blocks.residual_norm(h, norm=blocks.Norm("rms", P["n1"]))
    y = F.linear(blocks.dropout(F.linear(y, P["w1"]), p, state, relu=True), P["w2"])
    return blocks.residual_norm(y, h, norm=blocks.Norm("layer", P["n2"], P["b2"]), norm_in=blocks.Norm("rms", P["n1"]), gate=P["gate"], alpha=0.5, p=p, state=state,
                                return_sum=True)


def run_block(device, rows, width, table):
    """the operators together, as a block uses them: outputs against float64, every gradient against the float64 graph and against differences of it"""
    from lidarseg3d_amd import blocks
    gen = torch.Generator().manual_seed(rows)
    P = block_parameters(gen, width, table, device)
    tokens = indices(gen, table, (rows,), "few", device)
    state = blocks.DropoutState(17, device=device, step=1)
    p = 0.25
    y, s = block_forward(P, tokens, state, p)
    assert state.calls == 2
    dy, ds = tensor(gen, rows, width, device=device), tensor(gen, rows, width, device=device)
    grads = torch.autograd.grad([y, s], list(P.values()), [dy, ds])
    # the same block in float64 with the masks of the definition
    k1, inv = keep_mask(rows, 2 * width, p, 17, 1, 0)
    k2, _ = keep_mask(rows, width, p, 17, 1, 1)

    def plain(Q):
        rms = lambda v, w: v * torch.rsqrt(v.square().mean(1, keepdim=True) + 1e-5) * w
        h = 2.0 * Q["table"][tokens.cpu()]
        m = (torch.relu(rms(h, Q["n1"]) @ Q["w1"].t()) * k1 * inv) @ Q["w2"].t()
        t = 0.5 * h + Q["gate"] * (rms(m, Q["n1"]) * k2 * inv)
        d = t - t.mean(1, keepdim=True)
        return d * torch.rsqrt(d.square().mean(1, keepdim=True) + 1e-5) * Q["n2"] + Q["b2"], t
    Q = {k: v.detach().cpu().double().requires_grad_() for k, v in P.items()}
    yr, sr = plain(Q)
    want = torch.autograd.grad([yr, sr], list(Q.values()), [dy.cpu().double(), ds.cpu().double()])
    # products of `width` / 2 width terms in 32 bits come in between: K32 with the largest value of the tensor as scale, 8-fold for the five operators in a row
    for name, g, w in [("y", y, yr), ("s", s, sr)] + [("d " + n, g, w) for n, g, w in zip(P, grads, want)]:
        check(g, w.detach(), float(w.detach().abs().max()), what=name, k=8 * K32)
    # differences of the float64 block along a random direction: the derivative is the gradients' product with it
    dirs = {k: torch.randn(v.shape, generator=gen, dtype=torch.float64) for k, v in Q.items()}
    val = lambda e: sum(float((o * w.cpu().double()).sum()) for o, w in zip(plain({k: Q[k].detach() + e * dirs[k] for k in Q}), (dy, ds)))
    slope, along = (val(1e-6) - val(-1e-6)) / 2e-6, sum(float((g.cpu().double() * dirs[k]).sum()) for k, g in zip(Q, grads))
    assert abs(slope - along) <= 1e-4 * sum(float((g.cpu().double() * dirs[k]).abs().sum()) for k, g in zip(Q, grads))


def run_decoder(device, points, p, monkeypatch, frames=2, classes=17):
    """the SF-Phase decoder's training forward on the block operators against its torch composition with the same masks: F.dropout of the composition is
    given the operators' draws (same step, same order of calls)"""
    from lidarseg3d_amd import blocks, point_heads
    torch.manual_seed(1)
    m = point_heads.SemanticFeatureFusionModule(64, 48, 32, d_model=96, nhead=4, num_decoder_layers=2, dim_feedforward=192, dropout=p).to(device).train()
    for l in m.decoder.layers:  # the dropout of the class tokens' attention weights stays torch's in both forms
        l.self_attn.dropout = 0.0
    gen = torch.Generator().manual_seed(2)
    x = tensor(gen, points, 64, device=device).requires_grad_()
    e1, e2 = tensor(gen, frames, 48, classes, 1, device=device).requires_grad_(), tensor(gen, frames, 32, classes, 1, device=device).requires_grad_()
    batch = (torch.arange(points) * frames // points).float().to(device)
    dy = tensor(gen, points, 96, device=device)
    leaves = [x, e1, e2] + list(m.parameters())

    def run(state):
        blocks.use_in_training(m, state)
        y = m(x, e1, e2, batch, frames)
        return [y.detach()] + [g for g in torch.autograd.grad(y, leaves, [dy], allow_unused=True)]
    got = run(blocks.DropoutState(5, device=device, step=3))
    draws = blocks.DropoutState(5, device=device, step=3)
    monkeypatch.setattr(torch.nn.functional, "dropout", lambda t, q=0.5, training=True, inplace=False: blocks.dropout(t, q, draws) if training and q > 0 else t)
    want = run(None)
    assert len(got) == len(want)
    # The scale of a gradient is the largest gradient of any leaf, not its own: a key projection's bias moves all scores of a query alike, softmax does not see
    # it, and its gradient is an exact zero in the formulas: what is computed is the rounding of a sum whose terms (the keys' gradients, which also make up the
    # projection's weight gradient) are as large as the other leaves' and cancel.
    top = max(float(w.abs().max()) for w in want[1:] if w is not None)
    for i, (g, w) in enumerate(zip(got, want)):
        assert (g is None) == (w is None)
        if g is not None:
            # two float32 evaluations of the same formulas: 2 layers of 4 products (at most 192 terms), 3 norms each; K32 per norm and product
            rel = 2 * 2 * 7 * K32
            if i == 0 or points <= 1000:
                bound = rel * (float(w.abs().max()) if i == 0 else top)
                assert float((g - w).abs().max()) <= bound, (i, float((g - w).abs().max()), bound)
            elif w.dim() > 1:
                # Many points: a ReLU whose input is within its error of zero may open in one evaluation and not in the other, and an element of a gradient then
                # jumps.  The inputs a (LayerNorm rows times W1, entries +-1 / sqrt(96): deviation 0.58, density at most 0.4 / 0.58, |a| <= 3) are off by
                # at most rel / 2 * 3, so a share f <= 2 (rel / 2 * 3) 0.7 of the gates may differ; the hidden gradient's norm moves by sqrt(f), twice
                # for two layers.  (A wrong mask at p = 0.1 moves it by sqrt(0.18) = 0.42.)
                f = 2 * (rel / 2 * 3) * 0.7
                assert float((g - w).norm()) <= (rel + 2 * f ** 0.5) * float(w.norm()), (i, float((g - w).norm() / w.norm()))


def run_reader(device, voxels):
    """the TransVFE reader's training forward on the block operators against its torch composition (no dropout there)"""
    from lidarseg3d_amd import blocks, readers
    torch.manual_seed(3)
    m = readers.TransformerVoxelFeatureExtractor(num_input_features=5, num_layers=2).to(device).train()
    gen = torch.Generator().manual_seed(4)
    v, n = tensor(gen, voxels, 5, 5, device=device), (torch.arange(voxels) % 5 + 1).to(torch.int32).to(device)
    res = []
    for state in (None, blocks.DropoutState(1, device=device)):
        y = blocks.use_in_training(m, state)(v, n)
        res.append([y.detach()] + list(torch.autograd.grad(y, list(m.parameters()), [torch.ones_like(y)])))
    for w, g in zip(*res):
        assert float((g - w).abs().max()) <= 2 * 2 * 6 * K32 * max(float(w.abs().max()), 1e-3), (float((g - w).abs().max()), float(w.abs().max()))


def run_camera_sampling(device, points):
    """the camera features at the points as one weighted lookup against eight gathers: the same products added in the same order, and the maps' gradient
    against float64"""
    from lidarseg3d_amd import point_heads
    gen = torch.Generator().manual_seed(6)
    img = tensor(gen, 2, 3, 48, 9, 13, device=device).requires_grad_()
    cuv = torch.cat([torch.ones(points, 1), torch.randint(0, 3, (points, 1), generator=gen).float() - 1.0, torch.rand(points, 2, generator=gen) * 2.4 - 1.2], 1).to(device)
    bidx = (torch.arange(points) * 2 // points).float().to(device)
    want, got = point_heads._sample_image_rows(img, cuv, bidx), point_heads._sample_image_rows(img, cuv, bidx, lookup=True)
    check(got, want.detach().cpu().double(), got.detach().cpu().double().abs().amax(1, keepdim=True) + 1.0, what="sampled features")
    dy = tensor(gen, points, 48, device=device)
    (g,) = torch.autograd.grad(got, [img], [dy])
    i64 = img.detach().cpu().double().requires_grad_()
    w64 = point_heads._sample_image_rows(i64, cuv.cpu(), bidx.cpu())
    (ref,) = torch.autograd.grad(w64, [i64], [dy.cpu().double()])
    (mag,) = torch.autograd.grad(point_heads._sample_image_rows(i64, cuv.cpu(), bidx.cpu()), [i64], [dy.cpu().double().abs()])
    check(g, ref, mag, what="d maps", k=(points + 16) * 2.0 ** -24)


def run_use_in_training(device):
    """use_in_training reaches the decoder, the reader and the heads' dropout, keeps the parameters' names, and state None undoes it"""
    from lidarseg3d_amd import blocks, build_detector, models_cfg
    model = build_detector(models_cfg.mseg3d(), train_cfg=None, test_cfg={}).to(device).train()
    names = list(model.state_dict())
    state = blocks.DropoutState(1, device=device)
    assert blocks.use_in_training(model, state) is model
    assert list(model.state_dict()) == names and model.point_head.block_state is state and model.point_head.sffm.block_state is state
    drops = [m for m in model.modules() if isinstance(m, torch.nn.Dropout)]
    assert drops and all(type(m) is blocks.Dropout and m.state is state and m.training for m in drops)
    x = torch.ones(40, 32, device=device)
    y = drops[0](x)
    assert state.calls == 1 and 0 < int((y == 0).sum()) < y.numel() and torch.equal(drops[0].eval()(x), x)
    blocks.use_in_training(model, None)
    assert model.point_head.block_state is None and all(m.state is None for m in drops)


def run_checkpointing(device, reentrant):
    import pytest
    from torch.utils.checkpoint import checkpoint

    from lidarseg3d_amd import blocks
    torch.manual_seed(5)
    x, r, w = (torch.randn(s).to(device).requires_grad_() for s in ((37, 24), (37, 24), (24,)))
    dy = torch.randn(37, 24).to(device)
    state = blocks.DropoutState(11, device=device)

    def block(x, r, calls=(None, None)):
        h = blocks.dropout(x, 0.3, state, call=calls[0], relu=True)
        return blocks.residual_norm(h, r, norm=blocks.Norm("rms", w, None, 1e-5), p=0.2, state=state, call=calls[1])

    y = block(x, r)
    want = torch.autograd.grad(y, (x, r, w), dy)
    state.calls = 0
    for t in (x, r, w):
        t.grad = None
    z = checkpoint(block, x, r, (0, 1), use_reentrant=reentrant)
    z.backward(dy)
    assert torch.equal(y, z) and all(torch.equal(t.grad, g) for t, g in zip((x, r, w), want))
    z = checkpoint(block, x, r, use_reentrant=reentrant)
    assert torch.equal(y, z)
    with pytest.raises(RuntimeError, match="activation checkpointing"):
        z.backward(dy)
    assert state.calls == 2
    torch.autograd.grad(block(x, r), (x, r, w), dy)  # the engine is none the worse


def run_accumulated_gradients(device):
    """.grad of leaves of one, two and three dimensions over two backward passes: twice the single gradient, in memory of its own for each leaf, whatever x and the
    residual share inside (a plain sum has one gradient for both)"""
    from lidarseg3d_amd import blocks
    gen = torch.Generator().manual_seed(31)
    for shape in ((24,), (5, 24), (2, 3, 24)):
        for norm in (None, blocks.Norm("layer")):
            x, r = (tensor(gen, *shape, device=device).requires_grad_() for _ in range(2))
            dy = tensor(gen, *shape, device=device)
            f = lambda: blocks.residual_norm(x, r, norm=norm)
            once = torch.autograd.grad(f(), [x, r], [dy])
            for _ in range(2):
                f().backward(dy)
            assert x.grad.data_ptr() != r.grad.data_ptr(), shape
            for t, g in zip((x, r), once):
                assert t.grad.shape == t.shape and torch.equal(t.grad, 2 * g), shape
        # both leaves through other operators, and a leaf that is x and residual at once
        x, r = (tensor(gen, *shape, device=device).requires_grad_() for _ in range(2))
        blocks.residual_norm(2 * x, 4 * r).backward(dy)
        assert torch.equal(x.grad, 2 * dy) and torch.equal(r.grad, 4 * dy)
        x.grad = None
        for _ in range(2):
            blocks.residual_norm(x, x).backward(dy)
        assert torch.equal(x.grad, 4 * dy)


def run_weight_gradient_of_no_columns(device):
    """a table without columns: the weights' gradient is a product over nothing, zeros in memory that held something else before"""
    from lidarseg3d_amd import blocks
    for T in (F32, BF16):
        for ix in (torch.tensor([[1, 1], [0, 4], [-1, 9]]), torch.zeros(2, 3, 700, dtype=torch.int64)):
            junk = [torch.full(ix.shape, 7.0, device=device) for _ in range(4)]
            del junk
            table, w = torch.zeros(5, 0, dtype=T, device=device, requires_grad=True), torch.rand(ix.shape).to(device).requires_grad_()
            y = blocks.embedding(table, ix.to(device), weight=w)
            assert y.shape == (*ix.shape[:-1], 0)
            dt, dw = torch.autograd.grad(y.sum(), [table, w])
            assert dt.shape == (5, 0) and torch.equal(dw, torch.zeros_like(w))


def operator_calls(device):
    """name -> a call of one input [4, 8] of each operator"""
    from lidarseg3d_amd import blocks
    st = blocks.DropoutState(1, device=device)
    ix, wt = torch.tensor([0, 3, 3], device=device), torch.ones(3, 2, device=device)
    return {"dropout": lambda x: blocks.dropout(x, 0.5, st.tensor, call=0), "relu dropout": lambda x: blocks.dropout(x, 0.5, st.tensor, call=0, relu=True),
            "residual_norm": lambda x: blocks.residual_norm(torch.ones_like(x), x, norm=blocks.Norm("layer"), p=0.5, state=st.tensor, call=1),
            "norm weight": lambda x: blocks.residual_norm(torch.ones(3, 8, device=device), norm=blocks.Norm("rms", x.sum(0))),
            "gate": lambda x: blocks.residual_norm(torch.ones(4, 8, device=device), gate=x),
            "embedding": lambda x: blocks.embedding(x, ix), "lookup weights": lambda x: blocks.embedding(torch.ones(5, 6, device=device), torch.zeros(4, 8, dtype=torch.int64, device=device), weight=x)}


def run_forward_mode(device):
    """a tangent is refused wherever it comes in - inputs, parameters, the gradients of a backward pass - and the calls work again afterwards"""
    import pytest
    import torch.autograd.forward_ad as fw
    for name, f in operator_calls(device).items():
        for wants_grad in (False, True):
            with fw.dual_level():
                x = torch.randn(4, 8).to(device).requires_grad_(wants_grad)
                with pytest.raises(RuntimeError, match="forward-mode"):
                    f(fw.make_dual(x, torch.ones_like(x)))
        x = torch.randn(4, 8).to(device).requires_grad_()
        y = f(x)
        with fw.dual_level():
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(y, [x], [fw.make_dual(torch.ones_like(y), torch.ones_like(y))], retain_graph=True)
            assert torch.isfinite(f(x)).all()  # no tangent: an ordinary call
        assert torch.isfinite(torch.autograd.grad(y, [x], [torch.ones_like(y)])[0]).all()


def run_tracers_and_wrapped_tensors(device):
    """torch.jit.trace, make_fx and fake tensors, torch.func's transforms, batched gradients: refused with the reason; ordinary calls work again afterwards, also under a
    dispatch mode that only looks on"""
    import warnings

    import pytest
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils._python_dispatch import TorchDispatchMode

    class Onlooker(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    for name, f in operator_calls(device).items():
        x = torch.randn(4, 8).to(device)
        want = f(x)
        for wants_grad in (False, True):
            leaf = x.clone().requires_grad_(wants_grad)
            with warnings.catch_warnings():
                warnings.simplefilter("ignore")
                with pytest.raises(RuntimeError, match="cannot be traced"):
                    torch.jit.trace(f, leaf, check_trace=False)
            for mode in ("real", "fake"):
                with pytest.raises(RuntimeError, match="cannot be traced"):
                    make_fx(f, tracing_mode=mode, _allow_non_fake_inputs=True)(leaf)
        with FakeTensorMode(allow_non_fake_inputs=True) as mode:
            fake = mode.from_tensor(x)
            with pytest.raises(RuntimeError, match="cannot be traced"):
                f(fake)
        for call in (lambda: f(fake), lambda: torch.func.vmap(f)(torch.stack([x, x])), lambda: torch.func.grad(lambda t: f(t).sum())(x),
                     lambda: torch.func.jvp(f, (x,), (x,)), lambda: torch.func.functionalize(f)(x)):
            with pytest.raises(RuntimeError, match="needs tensors in memory"):
                call()
        leaf = x.clone().requires_grad_()
        y = f(leaf)
        with pytest.raises(RuntimeError, match="needs tensors in memory"):
            torch.autograd.grad(y, [leaf], [torch.ones(2, *y.shape, device=device)], is_grads_batched=True, retain_graph=True)
        with Onlooker():
            assert torch.equal(f(x), want)
        assert torch.equal(f(x), want) and torch.isfinite(torch.autograd.grad(y, [leaf], [torch.ones_like(y)])[0]).all()


def run_converted_dropouts(device):
    """use_in_training keeps a dropout's identity: hooks, names that share one module, a bare nn.Dropout as the model, in-place work; None gives back nn.Dropout"""
    import copy

    from lidarseg3d_amd import blocks
    nn = torch.nn

    class Twice(nn.Module):
        def __init__(self):
            super().__init__()
            self.a = self.b = nn.Dropout(0.5)
            self.seq = nn.Sequential(nn.Identity(), self.a, nn.Dropout(0.25, inplace=True), nn.Dropout(0.25).eval())
            self.own = blocks.Dropout(0.5)

    class Special(nn.Dropout):
        pass
    m, seen = Twice(), []
    m.special = Special(0.5)
    before = dict(m.named_modules(remove_duplicate=False))
    m.a.register_forward_hook(lambda mod, i, o: seen.append("hook"))
    state, x = blocks.DropoutState(3, device=device), torch.ones(64, 32, device=device)
    blocks.use_in_training(m, state)
    assert all(mod is before[name] for name, mod in m.named_modules(remove_duplicate=False)) and m.a is m.b is m.seq[1] and isinstance(m.a, nn.Dropout)
    assert type(m.special) is Special and not m.seq[3].training and torch.equal(m.seq[3](x), x)
    y, z = m.a(x), m.b(x)
    assert state.calls == 2 and seen == ["hook", "hook"] and not torch.equal(y, z)
    assert torch.equal(y, blocks.dropout(x, 0.5, state.tensor, call=0)) and torch.equal(z, blocks.dropout(x, 0.5, state.tensor, call=1))
    t = x.clone()
    assert m.seq[2](t) is t and torch.equal(t, blocks.dropout(x, 0.25, state.tensor, call=2))
    t = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(m.seq[2](t * 1.0), [t], [torch.ones_like(t)])
    assert torch.equal(g, blocks.dropout(x, 0.25, state.tensor, call=3))
    other = copy.deepcopy(m)
    assert type(other.a) is blocks.Dropout and other.a is other.b
    blocks.use_in_training(m, None)
    assert type(m.a) is type(m.seq[2]) is nn.Dropout and m.seq[2].inplace and type(m.own) is blocks.Dropout and m.own.state is None
    torch.manual_seed(1)
    want = torch.nn.functional.dropout(x, 0.5, True)
    torch.manual_seed(1)
    assert torch.equal(m.a(x), want) and len(seen) == 3
    # again, another state in between; a dropout that is the whole model
    second = blocks.DropoutState(4, device=device)
    assert blocks.use_in_training(blocks.use_in_training(m, state), second).a.state is second and type(blocks.use_in_training(m, None).a) is nn.Dropout
    bare = nn.Dropout(0.5)
    assert blocks.use_in_training(bare, second) is bare and torch.equal(bare(x), blocks.dropout(x, 0.5, second.tensor, call=0))
    assert type(blocks.use_in_training(bare, None)) is nn.Dropout


def run_differentiated_evaluation(device, points):
    """modules in evaluation mode compute the torch composition bit for bit after use_in_training, gradients included"""
    from lidarseg3d_amd import blocks, point_heads, readers
    torch.manual_seed(6)
    gen = torch.Generator().manual_seed(7)
    decoder = point_heads.SemanticFeatureFusionModule(64, 48, 32, d_model=96, nhead=4, num_decoder_layers=1, dim_feedforward=192, dropout=0.3).to(device).eval()
    reader = readers.TransformerVoxelFeatureExtractor(num_input_features=5, num_layers=1).to(device).eval()
    x = tensor(gen, points, 64, device=device).requires_grad_()
    e1, e2 = tensor(gen, 2, 48, 9, 1, device=device), tensor(gen, 2, 32, 9, 1, device=device)
    batch = (torch.arange(points) * 2 // points).float().to(device)
    vox, num = tensor(gen, points, 5, 5, device=device), (torch.arange(points) % 5 + 1).to(torch.int32).to(device)
    forms = {"decoder": (decoder, lambda m: m._forward_train(x, e1, e2, batch, 2), [x] + list(decoder.parameters())),
             "reader": (reader, lambda m: m._forward_train(vox, num), list(reader.parameters()))}
    state = blocks.DropoutState(1, device=device)
    calls = []
    keep = blocks.residual_norm
    blocks.residual_norm = lambda *a, **k: (calls.append(1), keep(*a, **k))[1]
    try:
        for name, (m, f, leaves) in forms.items():
            res = []
            for s in (None, state):
                y = f(blocks.use_in_training(m, s))
                res.append([y.detach()] + list(torch.autograd.grad(y, leaves, [torch.ones_like(y)], allow_unused=True)))
                assert not calls, name
            if device == "cpu":  # (on the device a library product may add in another order; the operators are not called at all there, above)
                assert torch.equal(res[0][0], res[1][0]), name
            m.train()
            f(m)
            assert calls, name
            calls.clear()
            m.eval()
    finally:
        blocks.residual_norm = keep
    head = point_heads.PointSegMSeg3DHead
    assert head.block_state is None
    stub = type("M", (), {"block_state": state, "training": False})()
    assert blocks.training_state(stub) is None
    stub.training = True
    assert blocks.training_state(stub) is state and state.calls > 0


def run_dropped_rows_beside_infinities(device):
    """rows of infinities and NaN behind a norm, of which the mask leaves nothing, at widths that leave lanes without columns: such a row is its residual, its norm and
    the residual's gradient are those of a row of zeros"""
    from lidarseg3d_amd import blocks
    gen = torch.Generator().manual_seed(41)
    for c, p, T, R, gate_kind in ((1, 0.9, F32, F32, None), (7, 0.9, BF16, BF16, "channel"), (9, 0.9, F16, F32, None), (70, 0.99, F32, F32, "full"), (70, 0.99, BF16, F32, None),
                                  (100, 0.99, F32, F32, None), (523, 0.999, F32, F32, "channel"), (523, 0.999, F16, F16, None)):
        n = 60
        for kind in ("layer", "rms"):
            x = torch.full((n, c), float("inf"), dtype=T)
            x[::3, c // 2] = float("nan")
            x[1::3] = -x[1::3]
            r, dy = tensor(gen, n, c, dtype=R), tensor(gen, n, c, dtype=T)
            gate = {None: None, "channel": tensor(gen, c), "full": tensor(gen, n, c, dtype=T)}[gate_kind]
            norm_in, norm = (kind, tensor(gen, c), tensor(gen, c), 1e-5), ("layer", tensor(gen, c), None, 1e-5)
            keep, _ = keep_mask(n, c, p, 8, 0, 4)
            gone = ~keep.any(1)
            assert 5 <= int(gone.sum()) < n, (c, int(gone.sum()))
            put = lambda t: None if t is None else t.to(device)
            xd, rd = put(x).requires_grad_(), put(r).requires_grad_()
            mod = lambda m: blocks.Norm(m[0], put(m[1]), put(m[2]), m[3])
            y, s = blocks.residual_norm(xd, rd, norm=mod(norm), norm_in=mod(norm_in), gate=put(gate), alpha=0.5, p=p, state=blocks.DropoutState(8, device=device).tensor, call=4,
                                        return_sum=True)
            (dr,) = torch.autograd.grad(y, [rd], [put(dy)])
            ref = residual_norm_reference(torch.zeros_like(x), r, norm, norm_in, gate, 0.5, p, (8, 0, 4), dy, None)
            for name, got in (("y", y), ("s", s), ("residual", dr)):
                value, scale = ref[name]
                check(got.detach().cpu()[gone], value[gone], scale[gone], what="%s, c %d, %s" % (name, c, kind))


def run_rows_near_the_largest_value(device):
    """equal values near the type's largest at widths that leave lanes without columns: (0 - mean) / std overflows there and must not reach the row, its gradient or, through rows
    that a workgroup does not have, the parameters' gradients.  Values and widths are powers of two: mean and deviation are exact"""
    from lidarseg3d_amd import blocks
    gen = torch.Generator().manual_seed(43)
    n, eps = 5, 1e-5
    std = eps ** -0.5
    for T in (F32, BF16):
        for c in (1, 2, 4, 8, 16):
            x = torch.full((n, c), -2.0 ** 127, dtype=T, device=device).requires_grad_()
            w, b = (tensor(gen, c, device=device).requires_grad_() for _ in range(2))
            wi = tensor(gen, c, device=device).requires_grad_()
            dy = tensor(gen, n, c, dtype=T, device=device)
            # norm alone: y = b, dx = (u - mean u) / std with u = w dy, dw = 0, db = sum dy
            y = blocks.residual_norm(x, norm=blocks.Norm("layer", w, b, eps))
            dx, dw, db = torch.autograd.grad(y, [x, w, b], [dy])
            dyd = dy.cpu().double()
            u = dyd * w.detach().cpu().double()
            check(y, b.detach().cpu().double().expand(n, c), 0.0, what="y")
            check(dx, std * (u - u.mean(1, keepdim=True)), std * _rmax(u), what="dx")
            assert bool((dw == 0).all()), (T, c)
            check(db, dyd.sum(0), dyd.abs().sum(0), what="db")
            # behind another norm: t = 0, s = residual
            r = tensor(gen, n, c, dtype=T, device=device).requires_grad_()
            y, s = blocks.residual_norm(x, r, norm=blocks.Norm("rms", w, None, eps), norm_in=blocks.Norm("layer", wi, None, eps), return_sum=True)
            gx, gr, gw, gi = torch.autograd.grad([y, s], [x, r, w, wi], [dy, dy])
            assert torch.equal(s, r) and torch.isfinite(gx).all() and bool((gi == 0).all()), (T, c)
            ref = residual_norm_reference(torch.zeros(n, c), r, ("rms", w, None, eps), ("layer", wi, None, eps), None, 1.0, 0.0, None, dy, dy)
            check(y, *ref["y"], what="y behind a norm")
            check(gr, *ref["residual"], what="d residual")
            check(gw, *ref["w_out"], what="d weight")


def run_rows_of_equal_values(device):
    """rows of one value at widths that are no power of two: 2-byte values times up to 8192 add up exactly in 32 bits, so the deviation is 0, the norm is its bias and the
    gradient of its weight is 0; the type's lowest and highest values do not overflow on the way"""
    from lidarseg3d_amd import blocks
    for T in (BF16, F16, F32):
        for c in (1, 3, 17, 65, 96, 129, 517, 771, 1000, 4099, 8191):
            top = float(torch.finfo(T).max)
            values = torch.tensor([top, -top, 60000.0, 0.1, -0.1, 1.0 / 3.0, 0.0, float(torch.finfo(T).tiny)]).to(T if T != F32 else BF16).to(T)  # (f32: values of 8 bits, and its extremes)
            if T == F32:
                values[0], values[1] = 2.0 ** 127, -2.0 ** 127
            x = values.unsqueeze(1).expand(-1, c).contiguous().to(device)
            w, b = torch.full((c,), 2.0, device=device, requires_grad=True), torch.arange(float(c), device=device)
            for norm_in in (None, blocks.Norm("layer")):
                y = blocks.residual_norm(x, norm=blocks.Norm("layer", w, b.to(T)), norm_in=norm_in)
                assert torch.equal(y.detach(), b.to(T).expand_as(y)), (T, c)
                (dw,) = torch.autograd.grad(y, [w], [torch.ones_like(y)])
                assert bool((dw == 0).all()), (T, c)
    # a residual that leaves one value in every column
    x, r = torch.full((5, 771), 512.0, dtype=F16, device=device), torch.full((5, 771), 7.0, dtype=F16, device=device)
    assert bool((blocks.residual_norm(x, r, norm=blocks.Norm("layer"), alpha=-3.0) == 0).all())


def run_single_value_gates(device):
    """a gate of one value, of a 2-byte type: its gradient is one sum, rounded once.  Every channel's sum is 1 + h (1 - 2^-6), h half a step of the type at 1, and
    there are so many channels that the total lies near the upper one of two neighbours; channels rounded for themselves would be 1 each and the total the lower"""
    from lidarseg3d_amd import blocks
    for T, R, c, want in ((BF16, BF16, 257, 258.0), (BF16, F32, 257, 258.0), (F16, F16, 2049, 2050.0)):
        h = unit(T)
        x = torch.tensor([[1.0], [h * (1 - 2.0 ** -6)]], dtype=torch.float64).to(T).expand(2, c).contiguous().to(device)
        assert float(x.double().sum()) == c * (1 + h * (1 - 2.0 ** -6))
        for shape in ((1,), (), (1, 1)):
            g = torch.full(shape, 0.5, dtype=T, device=device, requires_grad=True)
            s = blocks.residual_norm(x, torch.zeros(2, c, dtype=R, device=device), gate=g)
            assert torch.equal(s, 0.5 * x.to(R))
            (dg,) = torch.autograd.grad(s, [g], [torch.ones(2, c, dtype=R, device=device)])
            assert dg.shape == g.shape and dg.dtype == T and float(dg) == want, (T, shape, float(dg))


def run_one_element_with_a_gate(device):
    """x of one element and a gate of one element in another type: a single value, as at any other size"""
    from lidarseg3d_amd import blocks
    for shape in ((1, 1), (1, 1, 1)):
        x, g = torch.full(shape, 3.0, dtype=BF16, device=device, requires_grad=True), torch.full(shape, 0.5, device=device, requires_grad=True)
        y = blocks.residual_norm(x, gate=g)
        dx, dg = torch.autograd.grad(y, [x, g], [torch.full(shape, 2.0, dtype=BF16, device=device)])
        assert float(y.detach()) == 1.5 and float(dx) == 1.0 and float(dg) == 6.0 and y.shape == dx.shape == dg.shape == shape


def run_camera_sampling_types(device):
    """camera maps of a 2-byte type (an image network in mixed precision) and of float64, coordinates of either: the lookup gives what the gathers give, in their type"""
    from lidarseg3d_amd import point_heads
    gen = torch.Generator().manual_seed(61)
    points = 50
    cuv = torch.cat([torch.ones(points, 1), torch.randint(0, 2, (points, 1), generator=gen).float() * 2 - 1.0, torch.rand(points, 2, generator=gen) * 2.4 - 1.2], 1).to(device)
    bidx = torch.zeros(points, device=device)
    for T, P in ((BF16, F32), (F16, F32), (F32, F32), (torch.float64, F32), (F32, torch.float64), (F32, F16), (F16, F16)):
        img = tensor(gen, 1, 2, 16, 5, 7, device=device).to(T).requires_grad_()
        want, got = (point_heads._sample_image_rows(img, cuv.to(P), bidx, lookup) for lookup in (False, True))
        assert got.dtype == want.dtype, (T, P)
        # eight products, added in the same order; a 2-byte sum of the gathers is rounded at every step
        assert float((got.double() - want.double()).abs().max()) <= (16 * unit(want.dtype) + K32) * float(img.detach().abs().max()), (T, P)
        dy = tensor(gen, points, 16, device=device).to(want.dtype)
        (g,) = torch.autograd.grad(got, [img], [dy])
        assert g.dtype == T, (T, P)
        if want.dtype == F32:  # the lookup: sums in 32 bits, rounded to the maps' type once; the gathers in float64 with the same weights as reference
            i64 = img.detach().cpu().double().requires_grad_()
            ref, mag = (torch.autograd.grad(point_heads._sample_image_rows(i64, cuv.cpu().to(P), bidx.cpu()), [i64], [d])[0] for d in (dy.cpu().double(), dy.cpu().double().abs()))
            check(g, ref, mag, what="d maps", k=(points + 16) * 2.0 ** -24)


def run_negated_views(device):
    """tensors whose memory holds the other sign (the imaginary part of a conjugate), contiguous and not, in every place of every operator, gradients among them"""
    from lidarseg3d_amd import blocks
    gen = torch.Generator().manual_seed(71)
    z = torch.complex(torch.randn(6, 1, generator=gen), torch.randn(6, 1, generator=gen)).to(device)
    for neg in (torch._neg_view(tensor(gen, 4, 8, device=device)), z.conj().imag):
        assert neg.is_neg()
        plain = neg.clone()
        assert not plain.is_neg()
        n, c = plain.shape
        st = blocks.DropoutState(1, device=device).tensor
        ix = torch.tensor([[0, 1, 1]] * n, device=device)
        o, wide = tensor(gen, n, c, device=device), tensor(gen, 9, c, device=device)
        weights = lambda t: t.expand(n, 3) if c < 3 else t[:, :3]
        vec = lambda t: torch._neg_view(t[0].neg()) if t.is_neg() else t[0]
        calls = [lambda t: blocks.dropout(t, 0.25, st, call=0), lambda t: blocks.dropout(t, 0.25, st, call=0, relu=True), lambda t: blocks.residual_norm(t, o, norm=blocks.Norm("layer")),
                 lambda t: blocks.residual_norm(o, t, norm=blocks.Norm("rms")), lambda t: blocks.residual_norm(o, t, gate=t), lambda t: blocks.residual_norm(o, gate=vec(t)),
                 lambda t: blocks.residual_norm(o, norm=blocks.Norm("layer", vec(t), vec(t)), norm_in=blocks.Norm("rms", vec(t))), lambda t: blocks.embedding(t, ix),
                 lambda t: blocks.embedding(wide, ix, weight=weights(t))]
        for i, f in enumerate(calls):
            res = []
            for t in (plain, neg):
                res.append(f(t))
                leaf = t.detach()
                assert leaf.is_neg() == t.is_neg()
                leaf.requires_grad_()
                y = f(leaf)
                dy = torch.ones_like(y)
                if t.is_neg():
                    dy = torch._neg_view(-dy)
                res += [y.detach(), torch.autograd.grad(y, [leaf], [dy])[0]]
            for a, b in zip(res[:3], res[3:]):
                assert torch.equal(a, b), i


# rows, c, type, index shape, weights, scale, how the tokens fall
EXACT_LOOKUP = [
    (1, 8, F32, (30000,), False, 1.0, "one"),          # one row over 3750 tiles of 8: the join looks for its end twice
    (3, 5, BF16, (52000,), False, 0.5, "few"),         # three rows of about 2170 tiles each
    (40, 3, F16, (9000, 2), True, 2.0, "empty"),       # two thirds of the entries name no row
    (9000, 9, F32, (20000,), False, 1.0, "text"),
    (70, 17, F32, (4097,), False, 1.0, "runs"),
    (11, 70, BF16, (1500, 3), True, 1.0, "few"),
]
# tiles of 16, 32 and 64 entries, more than 2^20 entries (eight to a thread in the sort), many long rows side by side, the camera maps' size
EXACT_LOOKUP_LARGE = [
    (700, 64, F32, (300000,), False, 1.0, "text"),
    (2, 64, BF16, (300007,), False, 0.5, "few"),
    (50, 128, F32, (300000,), False, 1.0, "uniform"),
    (5000, 130, F16, (100003, 3), True, 2.0, "empty"),
    (3, 64, F32, (1200000,), False, 1.0, "few"),
    (1, 64, F32, (1300001,), False, 1.0, "one"),
    (100000, 16, F16, (1100000,), False, 1.0, "uniform"),
    (32, 64, F32, (360000,), False, 1.0, "uniform"),
    (460800, 48, F32, (360000, 8), True, 1.0, "empty"),
    (32000, 1024, BF16, (16384,), False, 1.0, "text"),
    (3000000, 8, F32, (1500000,), False, 1.0, "text"),
]


def exact_indices(gen, rows, shape, how):
    n = int(np.prod(shape))
    if how == "one":
        ix = torch.full((n,), rows - 1)
    elif how == "text":  # frequency falling with rank: a few rows over many tiles, most over none
        ix = (rows ** torch.rand(n, generator=gen, dtype=torch.float64) - 1).long().clamp_(0, rows - 1)
    elif how == "runs":
        ix = torch.repeat_interleave(torch.arange(rows), torch.arange(rows) * 7 % 90 + 1)[:n]
        ix = torch.cat([ix, torch.zeros(n - ix.numel(), dtype=torch.int64)])[torch.randperm(n, generator=gen)]
    else:
        ix = torch.randint(0, min(rows, 3) if how == "few" else rows, (n,), generator=gen)
    if how == "empty":
        ix = torch.where(torch.rand(n, generator=gen) < 0.67, torch.randint(-2, 0, (n,), generator=gen), ix)
    return ix.reshape(shape)


def run_exact_lookup(case, device, seed=0, index=torch.int64):
    """whole numbers throughout: every product and sum is below 2^24 and exact in 32 bits in any order, so output and gradients equal those of integer arithmetic, rounded
    to their type once"""
    from lidarseg3d_amd import blocks
    rows, c, T, shape, weights, scale, how = case
    gen = torch.Generator().manual_seed(seed + rows + c)
    whole = lambda *s: torch.randint(-4, 5, s, generator=gen).to(device)
    ix = exact_indices(gen, rows, shape, how).to(device)
    n, k = ix.shape[0], ix.shape[1] if ix.dim() == 2 else 1
    table, dy = whole(rows, c), whole(n, c)
    wt = torch.randint(0, 3, shape, generator=gen).to(device) if weights else None
    padding = rows // 2 if rows > 20 else None
    t = table.to(T).requires_grad_()
    w = wt.float().requires_grad_() if weights else None
    y = blocks.embedding(t, ix.to(index), weight=w, scale=scale, padding_idx=padding)
    grads = torch.autograd.grad(y, [t] + ([w] if weights else []), [dy.to(T)])
    flat = ix.reshape(n, k)
    f = wt.reshape(n, k) if weights else torch.ones_like(flat)
    out, dt, dw = torch.zeros(n, c, dtype=torch.int64, device=device), torch.zeros(rows, c, dtype=torch.int64, device=device), torch.zeros_like(flat)
    mag = torch.zeros_like(dt)
    for j in range(k):
        at = torch.nonzero(flat[:, j] >= 0)[:, 0]
        row = table[flat[at, j]]
        out[at] += f[at, j].unsqueeze(1) * row
        dw[at, j] = (row * dy[at]).sum(1)
        if padding is not None:
            at = at[flat[at, j] != padding]
        term = f[at, j].unsqueeze(1) * dy[at]
        dt.index_add_(0, flat[at, j], term)
        mag.index_add_(0, flat[at, j], term.abs())
    assert int(mag.max()) < 2 ** 24, "the case is not exact"
    once = lambda v, type_: (v.double() * scale).to(torch.float32).to(type_)
    assert torch.equal(y.detach(), once(out, T)), case
    assert torch.equal(grads[0], once(dt, T)), (case, torch.nonzero(grads[0] != once(dt, T))[:4].tolist())
    if weights:
        assert torch.equal(grads[1], once(dw, F32).reshape(grads[1].shape)), case


def random_exact_lookup(rng, budget):
    """a case of at most `budget` values to add, its lengths spread over their logarithm"""
    log = lambda lo, hi: int(round(np.exp(rng.uniform(np.log(lo), np.log(max(lo, hi))))))
    c = log(1, 600)
    k = rng.choice([1, 1, 2, 5])
    n = log(1, max(1, min(1500000, budget // (c * k))))
    return (log(1, max(1, min(2000000, 4 * budget // c))), c, rng.choice([F32, BF16, F16]), (n,) if k == 1 else (n, k), k > 1, rng.choice([1.0, 0.5, 2.0]),
            rng.choice(["empty", "text", "few", "uniform"]) if n * k * 8 < 2 ** 24 else "empty")


def run_inputs_changed_before_the_backward_pass(device):
    """x, residual or gate changed in place after the forward pass: refused, whatever the number of dimensions the rows were made of"""
    import pytest

    from lidarseg3d_amd import blocks
    for shape in ((8,), (3, 8), (2, 3, 8)):
        for which in ("x", "residual", "gate"):
            w = torch.ones(8, device=device, requires_grad=True)
            t = {k: torch.ones(shape, device=device) for k in ("x", "residual", "gate")}
            y = blocks.residual_norm(t["x"], t["residual"], gate=t["gate"], norm=blocks.Norm("rms", w))
            t[which].add_(1)
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                y.sum().backward()
