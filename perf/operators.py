"""Cases and plain forms of the training-block operators of lidarseg3d_amd.blocks.

  dropout         y = keep * x / (1 - p) (optionally of relu(x)); the mask comes from a counter-based generator and is never stored
  residual_norm   t = norm_in(x);  s = alpha * residual + gate * dropout(t);  y = norm(s)      (every part but x optional)
  embedding       out[i] = scale * sum_k weight[i, k] * table[idx[i, k]];  gradient of the table by sorted tokens

`run` computes a pass in elementary torch operations, or (own = True) with the calls a user makes of lidarseg3d_amd.blocks.

The generator (all three parties compute the same draws): Philox4x32 with 10 rounds (Salmon, Moraes, Dror, Shaw: "Parallel random numbers:
as easy as 1, 2, 3", SC11), key = (low, high 32 bits of the seed), counter = (column / 8, row, call, step mod 2^32).  Its four output words
are eight 16-bit draws, the low half of a word first: one for each of the eight columns.  An element is dropped where its draw is below
round(65536 p); what is kept is scaled by 65536 / (65536 - round(65536 p)).
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}


# ------------------------------------------------------------------------------------------------------------------ cases
def _dropout(name, rows, c, dtype, p, relu=False):
    return {"name": name, "op": "dropout", "rows": rows, "c": c, "dtype": dtype, "p": p, "relu": relu}


def _norm(name, rows, c, dtype, stream=None, kind="layer", kind_in="", gate="", alpha=1.0, p=0.0, with_sum=False, train=True):
    """stream: type of the residual and of the sum; kind / kind_in: layer | rms | "" ; gate: "" | channel | full"""
    return {"name": name, "op": "residual_norm", "rows": rows, "c": c, "dtype": dtype, "stream": stream or dtype, "kind": kind, "kind_in": kind_in,
            "gate": gate, "alpha": alpha, "p": p, "with_sum": with_sum, "train": train}


def _embed(name, rows, k, table, c, dtype, spread, scale=1.0, weights=False, weight_grad=False, index="i64", train=True):
    """spread: zipf (text-like), uniform, image (bilinear corners in camera maps of 160 x 240 pixels, rows outside every camera empty)"""
    return {"name": name, "op": "embedding", "rows": rows, "k": k, "table": table, "c": c, "dtype": dtype, "spread": spread, "scale": scale,
            "weights": weights, "weight_grad": weight_grad, "index": index, "train": train}


def listed():
    return [
        # class-token embeddings of two frames (2 x 34 tokens, d_model 96): the smallest training call, launch latency counts
        _dropout("dropout_tokens", 68, 96, "f32", 0.1),
        # the decoder's feed-forward activation over two Waymo frames (2 x 180k points, ffn 192): the largest dropout of a training step
        _dropout("dropout_ffn_relu", 360000, 192, "f32", 0.1, relu=True),
        # an odd width in bf16: rows that start at every alignment
        _dropout("dropout_odd_bf16", 16411, 1001, "bf16", 0.25),
        # one token of a serving step, pre-norm of a residual stream in bf16
        _norm("norm_one_token", 1, 4096, "bf16", kind="rms", with_sum=True, train=False),
        # the decoder's post-norm over two Waymo frames: LayerNorm(residual + dropout(x)), d_model 96
        _norm("norm_decoder_f32", 360000, 96, "f32", p=0.1),
        # norms before and after a block with a channel gate and a scaled residual stream in f32, training
        _norm("norm_sandwich_mixed", 8192, 2048, "bf16", stream="f32", kind="rms", kind_in="rms", gate="channel", alpha=0.5, with_sum=True),
        # ragged sizes, a gate for each element, dropout, fp16
        _norm("norm_odd_gated_f16", 5003, 771, "f16", gate="full", alpha=1.25, p=0.2, with_sum=True),
        # a long prompt in serving: pre-norm with the running sum, no gradient
        _norm("norm_prompt_bf16", 16384, 4096, "bf16", kind="rms", with_sum=True, train=False),
        # eight tokens of a serving step looked up in a vocabulary
        _embed("embed_tokens_bf16", 8, 1, 32000, 4096, "bf16", "zipf", scale=64.0, train=False),
        # a training batch of text-like tokens, a few of them very frequent
        _embed("embed_vocab_bf16", 16384, 1, 32000, 1024, "bf16", "zipf", scale=32.0),
        # an embedding for each of the 32 beams of the scanner over two Waymo frames: few rows with very many tokens each
        _embed("embed_beams_f32", 360000, 1, 32, 64, "f32", "uniform", index="i32"),
        # camera features of two frames of six cameras ([2, 6, 48, 160, 240]) sampled at the points: 8 weighted rows for each, many of them empty
        _embed("embed_camera_f32", 360000, 8, 460800, 48, "f32", "image", weights=True, index="i32"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["dropout", "residual_norm", "residual_norm", "embedding", "embedding"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "dropout":
        c = _log(rng, 1, 8192)
        rows = _log(rng, 1, max(1, min(400000, 60000000 // c)))
        case = _dropout("", rows, c, dtype, rng.choice([0.05, 0.1, 0.25, 0.5, 0.9]), relu=rng.random() < 0.4)
    elif op == "residual_norm":
        c = rng.choice([32, 48, 64, 96, 128, 192, 256, 1024, 2048, 4096, 8192]) if rng.random() < 0.6 else _log(rng, 2, 8192)
        train = rng.random() < 0.65
        rows = _log(rng, 1, max(1, min(400000, 30000000 // c)))
        kind = rng.choice(["layer", "rms"])
        case = _norm("", rows, c, dtype, stream="f32" if rng.random() < 0.3 else dtype, kind=kind, kind_in=rng.choice(["", "", "layer", "rms"]),
                     gate=rng.choice(["", "", "channel", "full"]), alpha=rng.choice([1.0, 1.0, 0.5, 1.5]),
                     p=rng.choice([0.0, 0.1, 0.3]) if train else 0.0, with_sum=rng.random() < 0.5, train=train)
    else:
        c = rng.choice([32, 48, 64, 96, 256, 1024, 2048, 4096]) if rng.random() < 0.6 else _log(rng, 1, 4096)
        k = rng.choice([1, 1, 1, 3, 8])
        table = _log(rng, 2, max(2, min(300000, 60000000 // c)))
        rows = _log(rng, 1, max(1, min(300000, 60000000 // (c * k))))
        weights = k > 1 and rng.random() < 0.7
        train = rng.random() < 0.7
        case = _embed("", rows, k, table, c, dtype, rng.choice(["zipf", "uniform"]), scale=rng.choice([1.0, 1.0, 8.0]), weights=weights,
                      weight_grad=weights and train and rng.random() < 0.5, index=rng.choice(["i32", "i64"]), train=train)
    del case["name"]
    return case


# ------------------------------------------------------------------------------------------------------------------ inputs
def _zipf(table):
    w = 1.0 / (np.arange(table, dtype=np.float64) + 2.7)
    return w / w.sum()


def _image_entries(rows, table, gen, dev):
    """corner rows and weights of the points' bilinear samples: camera maps of h x w pixels stacked to `table` rows; -1 = no row"""
    h, w = 160, 240
    maps = table // (h * w)
    cam = torch.randint(0, maps, (rows,), generator=gen, device=dev)
    y = torch.rand(rows, generator=gen, device=dev) * (h + 1) - 1.0
    x = torch.rand(rows, generator=gen, device=dev) * (w + 1) - 1.0
    seen = torch.rand(rows, generator=gen, device=dev) < 0.7
    idx, wgt = [], []
    for corner in range(8):
        dm, dy, dx = corner & 1, (corner >> 1) & 1, (corner >> 2) & 1
        yy, xx = y.floor() + dy, x.floor() + dx
        g = (1 - (y - yy).abs()) * (1 - (x - xx).abs())
        ok = seen & (dm == 0) & (yy >= 0) & (yy < h) & (xx >= 0) & (xx < w)
        idx.append(torch.where(ok, (cam * h + yy.long().clamp(0, h - 1)) * w + xx.long().clamp(0, w - 1), torch.full_like(cam, -1)))
        wgt.append(torch.where(ok, g, torch.zeros_like(g)))
    return torch.stack(idx, 1), torch.stack(wgt, 1)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    T = _TYPES[case["dtype"]]

    def randn(*shape, scale=1.0, shift=0.0, dtype=T):
        return (torch.randn(*shape, generator=gen, device=dev) * scale + shift).to(dtype)

    s = {"case": case}
    if case["op"] != "embedding":
        # the dropout state of a training program: (seed, step) on the device, the number of the call within the step
        s["rng_host"] = (int(seed) * 2654435761 + 97 & 0x7FFFFFFFFFFFFFFF, 3 + int(seed) % 1000, 2 + int(seed) % 7)
        s["rng"] = torch.tensor(s["rng_host"][:2], dtype=torch.int64, device=dev)
    if case["op"] == "dropout":
        s["x"] = randn(case["rows"], case["c"]).requires_grad_()
        s["dy"] = randn(case["rows"], case["c"])
    elif case["op"] == "residual_norm":
        n, c, R = case["rows"], case["c"], _TYPES[case["stream"]]
        s["x"], s["residual"] = randn(n, c), randn(n, c, scale=2.0, dtype=R)
        for key in ("kind_in", "kind"):
            if case[key]:
                s[key] = [randn(c, scale=0.1, shift=1.0, dtype=R)] + ([randn(c, scale=0.1, dtype=R)] if case[key] == "layer" else [])
        if case["gate"]:
            s["gate"] = randn(c, scale=0.3, shift=0.5, dtype=R) if case["gate"] == "channel" else randn(n, c, scale=0.5, shift=0.5)
        s["leaves"] = [s["x"], s["residual"]] + s.get("kind_in", []) + s.get("kind", []) + ([s["gate"]] if case["gate"] else [])
        if case["train"]:
            for t in s["leaves"]:
                t.requires_grad_()
            s["dy"] = randn(n, c)
            if case["with_sum"]:
                s["ds"] = randn(n, c, dtype=R)
    else:
        n, k, V = case["rows"], case["k"], case["table"]
        wgt = None
        if case["spread"] == "image":
            idx, wgt = _image_entries(n, V, gen, dev)
        elif case["spread"] == "zipf":
            cdf = torch.from_numpy(np.cumsum(_zipf(V))).to(dev)
            rank = torch.searchsorted(cdf, torch.rand(n, k, generator=gen, device=dev, dtype=torch.float64)).clamp_(max=V - 1)
            idx = torch.randperm(V, generator=gen, device=dev)[rank]
        else:
            idx = torch.randint(0, V, (n, k), generator=gen, device=dev)
        if case["weights"] and wgt is None:
            wgt = torch.rand(n, k, generator=gen, device=dev)
        s["table"] = randn(V, case["c"])
        s["idx"] = (idx if k > 1 else idx[:, 0]).to(torch.int64 if case["index"] == "i64" else torch.int32).contiguous()
        s["weight"] = wgt
        if case["train"]:
            s["table"].requires_grad_()
            if case["weight_grad"]:
                wgt.requires_grad_()
            s["dy"] = randn(n, case["c"])
    return s


# ------------------------------------------------------------------------------------------------------------------ plain forms
def _keep(rows, c, p, rng, dev):
    """[rows, c] truth values and the factor of what is kept"""
    seed, step, call = rng
    thr = int(p * 65536 + 0.5)
    groups, low = (c + 7) // 8, 0xFFFFFFFF
    c0 = torch.arange(groups, device=dev, dtype=torch.int64).expand(rows, groups)
    c1 = torch.arange(rows, device=dev, dtype=torch.int64).unsqueeze(1).expand(rows, groups)
    c2, c3 = torch.full_like(c0, call & low), torch.full_like(c0, step & low)
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # 64-bit products; their upper halves are taken without the sign
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    draws = torch.stack([h for w in (c0, c1, c2, c3) for h in (w & 0xFFFF, w >> 16)], -1)
    keep = draws.reshape(rows, groups * 8)[:, :c] >= thr
    return keep, (65536.0 / (65536 - thr) if thr < 65536 else 0.0)


def _plain_norm(x, kind, params, eps):
    if kind == "layer":
        x = x - x.mean(1, keepdim=True)
    y = x * torch.rsqrt((x * x).mean(1, keepdim=True) + eps) * params[0]
    return y + params[1] if kind == "layer" else y


def _plain(s):
    case = s["case"]
    f32 = torch.float32
    if case["op"] == "dropout":
        keep, inv = _keep(case["rows"], case["c"], case["p"], s["rng_host"], s["x"].device)
        x = s["x"].detach().to(f32)
        if case["relu"]:
            keep = keep & (x > 0)
        zero = torch.zeros((), device=x.device)
        return [torch.where(keep, x * inv, zero).to(s["x"].dtype), torch.where(keep, s["dy"].to(f32) * inv, zero).to(s["x"].dtype)]
    if case["op"] == "residual_norm":
        train = case["train"]
        with torch.set_grad_enabled(train):
            # in 32 bits whatever the inputs' types; every result is rounded once, to its own type
            wide = [t.detach().to(f32).requires_grad_(train) for t in s["leaves"]]
            rest = wide[2:]
            x, residual = wide[:2]
            if case["kind_in"]:
                m = len(s["kind_in"])
                x, rest = _plain_norm(x, case["kind_in"], rest[:m], 1e-5), rest[m:]
            if case["p"] > 0:
                keep, inv = _keep(case["rows"], case["c"], case["p"], s["rng_host"], x.device)
                x = torch.where(keep, x * inv, torch.zeros((), device=x.device))
            m = len(s["kind"])
            if case["gate"]:
                x = x * rest[m]
            total = case["alpha"] * residual + x
            y = _plain_norm(total, case["kind"], rest[:m], 1e-5)
            outs = [y, total] if case["with_sum"] else [y]
            res = [o.detach().to(t.dtype) for o, t in zip(outs, (s["x"], s["residual"]))]
            if train:
                grads = torch.autograd.grad(outs, wide, [s["dy"].to(f32)] + ([s["ds"].to(f32)] if case["with_sum"] else []))
                res += [g.to(t.dtype) for g, t in zip(grads, s["leaves"])]
        return res
    table, idx = s["table"].detach(), s["idx"].to(torch.int64).reshape(case["rows"], case["k"])
    hit = (idx >= 0).unsqueeze(2)
    rows = torch.where(hit, table[idx.clamp(min=0)].to(f32), torch.zeros((), device=idx.device))
    wgt = s["weight"].detach().unsqueeze(2) if case["weights"] else None
    res = [((rows * wgt if case["weights"] else rows).sum(1) * case["scale"]).to(table.dtype)]
    if case["train"]:
        g = s["dy"].to(f32).unsqueeze(1) * case["scale"]
        if case["weight_grad"]:
            dw = (rows * g).sum(2)
        e = g * wgt if case["weights"] else g.expand_as(rows)
        # up to 10^5 tokens of one row: their sum in 64 bits
        at = torch.nonzero(idx.reshape(-1) >= 0)[:, 0]
        to, e = idx.reshape(-1)[at], e.reshape(-1, case["c"])[at].to(torch.float64)
        if case["table"] <= 64:  # a sum for each row: adding 10^4 tokens to one row one by one takes longer
            dt = torch.stack([(e * (to == v).unsqueeze(1)).sum(0) for v in range(case["table"])])
        else:
            dt = torch.zeros(table.shape, dtype=torch.float64, device=idx.device).index_add_(0, to, e)
        res.append(dt.to(table.dtype))
        if case["weight_grad"]:
            res.append(dw)
    return res


# ------------------------------------------------------------------------------------------------------------------ the framework's calls
def _own(s):
    from lidarseg3d_amd import blocks
    case = s["case"]
    if case["op"] == "dropout":
        y = blocks.dropout(s["x"], case["p"], s["rng"], call=s["rng_host"][2], relu=case["relu"])
        return [y, *torch.autograd.grad(y, [s["x"]], [s["dy"]])]
    if case["op"] == "residual_norm":
        norms = {}
        for key, arg in (("kind", "norm"), ("kind_in", "norm_in")):
            if case[key]:
                norms[arg] = blocks.Norm(case[key], *s[key], eps=1e-5)
        with torch.set_grad_enabled(case["train"]):
            out = blocks.residual_norm(s["x"], s["residual"], gate=s.get("gate"), alpha=case["alpha"], p=case["p"], state=s["rng"],
                                       call=s["rng_host"][2], return_sum=case["with_sum"], **norms)
        outs = list(out) if case["with_sum"] else [out]
        if not case["train"]:
            return outs
        return outs + list(torch.autograd.grad(outs, s["leaves"], [s["dy"]] + ([s["ds"]] if case["with_sum"] else [])))
    with torch.set_grad_enabled(case["train"]):
        y = blocks.embedding(s["table"], s["idx"], weight=s["weight"] if case["weights"] else None, scale=case["scale"], bag=case["k"] > 1)
    if not case["train"]:
        return [y]
    return [y, *torch.autograd.grad(y, [s["table"]] + ([s["weight"]] if case["weight_grad"] else []), [s["dy"]])]


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------------------------ the floor
def work(case):
    es = _SIZE[case["dtype"]]
    if case["op"] == "dropout":
        e = case["rows"] * case["c"]
        return {"bytes": 4 * e * es, "flops": 2 * e}
    if case["op"] == "residual_norm":
        n, c, rs = case["rows"], case["c"], _SIZE[case["stream"]]
        passes = 2 if case["train"] else 1  # x, residual in and y, sum out; backward: their gradients
        e = n * c
        b = passes * e * (2 * es + rs + (rs if case["with_sum"] else 0)) + (passes * e * es if case["gate"] == "full" else 0)
        per = 4 + (6 if case["kind_in"] else 0) + 8
        return {"bytes": b, "flops": e * per * (3 if case["train"] else 1)}
    n, k, V, c = case["rows"], case["k"], case["table"], case["c"]
    entries = n * k
    if case["spread"] == "image":
        entries = int(n * 0.7 * 4)
    used = float((1.0 - np.exp(-entries * _zipf(V))).sum()) if case["spread"] == "zipf" else V * (1.0 - math.exp(-entries / V))
    b = used * c * es + n * c * es + n * k * (8 if case["index"] == "i64" else 4) + (n * k * 4 if case["weights"] else 0)
    if case["train"]:
        b += n * c * es + V * c * es + (n * k * 4 if case["weight_grad"] else 0)
    return {"bytes": int(b), "flops": 2 * entries * c * (1 + (1 if case["train"] else 0) + (1 if case["weight_grad"] else 0))}


# ------------------------------------------------------------------------------------------------------------------ 64 bits, from the definitions
def _exact_mask(rows, c, p, rng):
    """element (r, j) is kept where its 16-bit draw reaches the threshold: numpy, unsigned 64-bit arithmetic, one draw column at a time"""
    seed, step, call = rng
    m32, u = np.uint64(0xFFFFFFFF), np.uint64
    g = (c + 7) // 8
    x = [np.broadcast_to(np.arange(g, dtype=u), (rows, g)), np.broadcast_to(np.arange(rows, dtype=u)[:, None], (rows, g)),
         np.full((rows, g), call % 2 ** 32, u), np.full((rows, g), step % 2 ** 32, u)]
    for r in range(10):
        key = (u((seed + r * 0x9E3779B9) % 2 ** 32), u(((seed >> 32) + r * 0xBB67AE85) % 2 ** 32))
        left, right = u(0xD2511F53) * x[0], u(0xCD9E8D57) * x[2]
        x = [(right >> u(32)) ^ x[1] ^ key[0], right & m32, (left >> u(32)) ^ x[3] ^ key[1], left & m32]
    thr = math.floor(65536 * p + 0.5)
    keep = np.empty((rows, g, 8), np.bool_)
    for j in range(8):
        keep[:, :, j] = ((x[j // 2] >> u(16 * (j % 2))) & u(0xFFFF)) >= u(thr)
    return torch.from_numpy(np.ascontiguousarray(keep.reshape(rows, g * 8)[:, :c])), (0.0 if thr >= 65536 else 65536.0 / (65536.0 - thr))


def _exact_stats(v, kind):
    mean = v.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(v[:, :1])
    return mean, 1.0 / ((v - mean).square().mean(1, keepdim=True) + 1e-5).sqrt()


def _exact_norm_back(u, hat, rstd, kind):
    r = u - hat * (u * hat).mean(1, keepdim=True)
    return rstd * (r - u.mean(1, keepdim=True) if kind == "layer" else r)


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        d = {k: v.detach().double() for k, v in s.items() if torch.is_tensor(v) and v.is_floating_point()}
        if case["op"] == "dropout":
            keep, inv = _exact_mask(case["rows"], case["c"], case["p"], s["rng_host"])
            f = keep.to(d["x"].device).double() * inv
            if case["relu"]:
                f = f * (d["x"] > 0)
            return [d["x"] * f, d["dy"] * f]
        if case["op"] == "residual_norm":
            x, kin, kout = d["x"], case["kind_in"], case["kind"]
            p_in, p_out = [[t.detach().double() for t in s.get(key, [])] for key in ("kind_in", "kind")]
            gate = d["gate"] if case["gate"] else torch.ones_like(x[:1])
            t = x
            if kin:
                mi, ri = _exact_stats(x, kin)
                hat_in = (x - mi) * ri
                t = hat_in * p_in[0] + (p_in[1] if kin == "layer" else 0.0)
            f = torch.ones_like(x[:1])
            if case["p"] > 0:
                keep, inv = _exact_mask(case["rows"], case["c"], case["p"], s["rng_host"])
                f = keep.to(x.device).double() * inv
            total = case["alpha"] * d["residual"] + gate * (t * f)
            mo, ro = _exact_stats(total, kout)
            hat = (total - mo) * ro
            res = [hat * p_out[0] + (p_out[1] if kout == "layer" else 0.0)]
            if case["with_sum"]:
                res.append(total)
            if not case["train"]:
                return res
            g = _exact_norm_back(d["dy"] * p_out[0], hat, ro, kout)
            if case["with_sum"]:
                g = g + d["ds"]
            dt = g * gate * f
            dx = _exact_norm_back(dt * p_in[0], hat_in, ri, kin) if kin else dt
            res += [dx, case["alpha"] * g]
            if kin:
                res += [(dt * hat_in).sum(0)] + ([dt.sum(0)] if kin == "layer" else [])
            res += [(d["dy"] * hat).sum(0)] + ([d["dy"].sum(0)] if kout == "layer" else [])
            if case["gate"]:
                dg = g * (t * f)
                res.append(dg.sum(0) if case["gate"] == "channel" else dg)
            return res
        idx = s["idx"].long().reshape(case["rows"], case["k"])
        out = torch.zeros(case["rows"], case["c"], dtype=torch.float64, device=idx.device)
        dt, dw = torch.zeros_like(d["table"]), torch.zeros(idx.shape, dtype=torch.float64, device=idx.device)
        for j in range(case["k"]):
            at = torch.nonzero(idx[:, j] >= 0)[:, 0]
            w = d["weight"][at, j].unsqueeze(1) * case["scale"] if case["weights"] else torch.full((1, 1), case["scale"], dtype=torch.float64, device=idx.device)
            row = d["table"][idx[at, j]]
            out[at] += w * row
            if case["train"]:
                dt.index_add_(0, idx[at, j], w * d["dy"][at])
                dw[at, j] = case["scale"] * (row * d["dy"][at]).sum(1)
        return [out] + ([dt] if case["train"] else []) + ([dw] if case["weight_grad"] else [])
