"""The work that the speed of the row norms, the grouped products and the optimiser's step is measured on.

A case is one pass through one operator as a program calls it: a norm of rows (with its gradients, or with an output in
8 bits), a product of ragged groups of rows with each group's own weights (with its gradients, or on 8-bit rows), or one
step of AdamW over all tensors of a network.  `listed()` gives the named cases, `draw(rng)` one more of the same ranges.

Sizes: rows are the active sites of a scene or the tokens of a batch, from a handful to the sites of several rooms; planes are
those of the package's networks (16 to 224) and of wide per-point blocks (up to 8192).  The optimiser's tensors are those of
the package's U-Net of seven levels and of its handwriting network, and the weights of a block of grouped products.
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
E4M3_MOST = 448.0
BLOCK = 256                                   # values that share a scale in an 8-bit state
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}
LR, BETA1, BETA2, EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 0.01
STEPS_DONE = 100                              # the optimiser has run for a while
NORM_EPS = 1e-6


def listed():
    return [
        # One call of a classifier's head on a handful of rows: the launch is all there is.
        dict(name="norm_few_rows", kind="norm", rows=7, planes=2048, type="bfloat16", residual=True, quantized=False, train=False),
        # A residual block over the sites of one room in training, the U-Net's third level's planes, fp32 as the convolutions
        # around it.
        dict(name="norm_room_train", kind="norm", rows=267011, planes=96, type="float32", residual=True, quantized=False, train=True),
        # A wide per-point block in training.
        dict(name="norm_wide_train", kind="norm", rows=16381, planes=4096, type="bfloat16", residual=True, quantized=False, train=True),
        # The same in serving, in front of a product on 8-bit rows.
        dict(name="norm_wide_8bit", kind="norm", rows=32768, planes=4096, type="bfloat16", residual=True, quantized=True, train=False),
        # Serving a small request: a few rows for each of eight groups, bound by the weights.
        dict(name="group_few_rows", kind="group", rows=37, groups=8, nin=1024, nout=1024, type="bfloat16", bias=False, quantized=False, train=False),
        # Rooms of sixteen sources with a layer of their own each, in the package's fp32, with gradients.
        dict(name="group_rooms_train", kind="group", rows=131071, groups=16, nin=64, nout=96, type="float32", bias=True, quantized=False, train=True),
        # A wide block in training: thirty-two groups, some of them empty, some large.
        dict(name="group_wide_train", kind="group", rows=32749, groups=32, nin=2048, nout=2048, type="bfloat16", bias=False, quantized=False, train=True),
        # Serving in 8 bits, many rows.
        dict(name="group_wide_8bit", kind="group", rows=65536, groups=16, nin=4096, nout=2048, type="bfloat16", bias=True, quantized=True, train=False),
        # The handwriting network's fifteen small tensors: latency.
        dict(name="step_strokes", kind="step", net="strokes", width=16, bits=32, grads="float32", copies=False),
        # The U-Net's tensors, states in 32 bits.
        dict(name="step_unet_32bit", kind="step", net="unet", width=32, bits=32, grads="float32", copies=False),
        # The same in 8 bits.
        dict(name="step_unet_8bit", kind="step", net="unet", width=32, bits=8, grads="float32", copies=False),
        # Grouped weights held in fp32 with the bf16 copies that the products read, bf16 gradients, 8-bit states.
        dict(name="step_groups_8bit", kind="step", net="groups", width=1024, bits=8, grads="bfloat16", copies=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "group", "group", "step"])
    if kind == "norm":
        planes = rng.choice([_log_int(rng, 16, 8192), 8 * _log_int(rng, 2, 1024)])
        quantized = rng.random() < 0.3
        return dict(kind=kind, rows=_log_int(rng, 1, min(400000, 134217728 // planes)), planes=planes,
                    type=rng.choice(["float32", "bfloat16", "bfloat16", "float16"]), residual=rng.random() < 0.7,
                    quantized=quantized, train=not quantized and rng.random() < 0.5)
    if kind == "group":
        quantized = rng.random() < 0.3
        nin, nout = (rng.choice([_log_int(rng, 16, 2048), 16 * _log_int(rng, 1, 128)]) for _ in range(2))
        rows = _log_int(rng, 1, min(200000, 60000000 // max(nin, nout)))
        return dict(kind=kind, rows=rows, groups=_log_int(rng, 1, min(64, 60000000 // (nin * nout))), nin=nin, nout=nout,
                    type="bfloat16" if quantized else rng.choice(["float32", "bfloat16", "bfloat16", "float16"]),
                    bias=rng.random() < 0.5, quantized=quantized, train=not quantized and rng.random() < 0.5)
    net = rng.choice(["strokes", "unet", "unet", "groups"])
    width = {"strokes": rng.randint(8, 32), "unet": rng.randint(8, 40), "groups": _log_int(rng, 64, 1024)}[net]
    return dict(kind=kind, net=net, width=width, bits=rng.choice([32, 8]), grads=rng.choice(["float32", "bfloat16"]),
                copies=rng.random() < 0.4)


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEVICE)


def _group_sizes(case, seed):
    """Ragged: log-normal shares, about every eighth group empty."""
    r = np.random.RandomState(seed % (1 << 31))
    share = np.exp(r.standard_normal(case["groups"])) * (r.random_sample(case["groups"]) > 0.125)
    if not share.any():
        share[r.randint(case["groups"])] = 1.0
    edges = np.floor(np.cumsum(share) / share.sum() * case["rows"] + 0.5).astype(np.int64)
    edges[-1] = case["rows"]
    return np.concatenate([[0], np.minimum(edges, case["rows"])])


def _tensor_sizes(case):
    """Numbers of values of a network's tensors."""
    w = case["width"]
    if case["net"] == "strokes":      # four levels of two submanifold layers of 3 x 3 with their norms, a class head
        sizes, nin = [], 1
        for nout in (w, 2 * w, 3 * w, 4 * w):
            sizes += [9 * nin * nout, nout, nout]
            nin = nout
        return sizes + [nin * 183, 183]
    if case["net"] == "unet":         # seven levels of w, 2 w .. 7 w planes, two layers each on the way down and up
        planes = [w * (i + 1) for i in range(7)]
        sizes = [27 * 3 * w]
        for i, p in enumerate(planes):
            sizes += [p, p, 27 * p * p] * 2
            if i < 6:
                sizes += [p, p, 8 * p * planes[i + 1], planes[i + 1], planes[i + 1], 8 * planes[i + 1] * p]
                sizes += [2 * p, 2 * p, 27 * 2 * p * p, p, p, 27 * p * p]
        return sizes + [w, w, w * 20, 20]
    return [w, 32 * w * w, 32 * w, 32 * w * w, 32 * w] + [w + 1, 16 * (w - 1) * w]  # a block of grouped products and odd ones


def prepare(case, seed):
    g = _generator(seed)
    if case["kind"] == "norm":
        n, c, t = case["rows"], case["planes"], TYPES[case["type"]]
        st = {"x": _normal(g, n, c).to(t), "residual": (3 * _normal(g, n, c)).to(t) if case["residual"] else None,
              "weight": 1 + 0.2 * _normal(g, c)}
        if case["train"]:
            st["d_out"], st["d_sum"] = _normal(g, n, c).to(t), _normal(g, n, c).to(t) if case["residual"] else None
            st["x"].requires_grad_()
            st["weight"].requires_grad_()
    elif case["kind"] == "group":
        n, t = case["rows"], TYPES[case["type"]]
        edges = _group_sizes(case, seed)
        sizes = np.diff(edges)
        st = {"offsets": torch.from_numpy(edges).to(DEVICE), "longest": int(sizes.max()),
              "bias": _normal(g, case["groups"], case["nout"]).to(t) if case["bias"] else None}
        x = _normal(g, n, case["nin"])
        w = _normal(g, case["groups"], case["nin"], case["nout"]) / math.sqrt(case["nin"])
        if case["quantized"]:          # rows as the norm leaves them, weights scaled once for each group and output plane
            st["scale"] = x.abs().amax(1).clamp_min(1e-30) / E4M3_MOST
            st["x"] = (x / st["scale"][:, None]).to(torch.float8_e4m3fn)
            st["weight_scale"] = w.abs().amax(1).clamp_min(1e-30) / E4M3_MOST
            st["weight"] = (w / st["weight_scale"][:, None, :]).transpose(1, 2).contiguous().to(torch.float8_e4m3fn)
        else:
            st["x"], st["weight"] = x.to(t), w.to(t)
            if case["train"]:
                st["d_out"] = _normal(g, n, case["nout"]).to(t)
                for k in ("x", "weight", "bias"):
                    if st[k] is not None:
                        st[k].requires_grad_()
    else:
        # Tensors are views of flat buffers, each at a whole number of blocks, as buckets for an all-reduce are laid out.
        sizes = _tensor_sizes(case)
        starts = np.concatenate([[0], np.cumsum([-(-s // BLOCK) for s in sizes])])
        total = int(starts[-1]) * BLOCK
        inside = torch.zeros(total, device=DEVICE)
        for s, a in zip(sizes, starts):
            inside[int(a) * BLOCK:int(a) * BLOCK + s] = 1
        grad = _normal(g, total) * inside * 1e-2
        first = _normal(g, total) * inside * 3e-3
        root = (_normal(g, total) * inside).abs() * 1e-2 + 1e-4 * inside
        flat = {"param": 0.05 * _normal(g, total) * inside, "grad": grad.to(TYPES[case["grads"]])}
        if case["bits"] == 8:
            for k, v in (("exp_avg", first), ("exp_avg_sq", root)):
                scale = v.view(-1, BLOCK).abs().amax(1).clamp_min(1e-30) / E4M3_MOST
                flat[k] = (v.view(-1, BLOCK) / scale[:, None]).to(torch.float8_e4m3fn).view(-1)
                flat[k + "_scale"] = scale
        else:
            flat["exp_avg"], flat["exp_avg_sq"] = first, root * root
        if case["copies"]:
            flat["copy"] = flat["param"].to(torch.bfloat16)
        st = {"flat": flat, "step": torch.tensor([STEPS_DONE], device=DEVICE), "seed": int(seed) % 65536}

        def views(k):
            per = BLOCK if not k.endswith("scale") else 1
            return [flat[k][int(a) * per:int(a) * per + (s if per > 1 else -(-s // BLOCK))] for s, a in zip(sizes, starts)]

        st["lists"] = {k: views(k) for k in flat}
    return dict(st, case=case)


# ---- the operators in plain form --------------------------------------------------------------------------------------

def _plain_norm(st):
    case, x = st["case"], st["x"].detach()
    s = (x.float() + st["residual"].float()).to(x.dtype) if case["residual"] else x
    f, w = s.float(), st["weight"].detach()
    k = torch.rsqrt((f * f).mean(1, keepdim=True) + NORM_EPS)
    h = f * k
    y = h * w
    if case["quantized"]:
        most = y.abs().amax(1, keepdim=True).clamp_min(1e-30)
        out = [(y * (E4M3_MOST / most)).clamp(-E4M3_MOST, E4M3_MOST).to(torch.float8_e4m3fn), most[:, 0] / E4M3_MOST]
    else:
        out = [y.to(x.dtype)]
    if case["residual"]:
        out.append(s)
    if case["train"]:
        d = st["d_out"].float()
        t = d * w
        dx = k * (t - h * (t * h).mean(1, keepdim=True))
        if case["residual"]:
            dx = dx + st["d_sum"].float()
        out += [dx.to(x.dtype), (d * h).sum(0)]
    return out


def _by_group(st, rows, longest):
    """Rows of the groups as [groups, longest, planes] in 32 bits, zeros behind a group's last row."""
    place = st["offsets"][:-1, None] + torch.arange(longest, device=DEVICE)
    real = place < st["offsets"][1:, None]
    return rows.float()[place.clamp_max(len(rows) - 1)] * real[:, :, None]


def _plain_group(st):
    case, x, w = st["case"], st["x"].detach(), st["weight"].detach()
    t, longest = TYPES[case["type"]], st["longest"]
    row = torch.arange(len(x), device=DEVICE)
    group = torch.searchsorted(st["offsets"], row, right=True) - 1
    place = row - st["offsets"][group]
    w = w.float().transpose(1, 2) if case["quantized"] else w.float()
    xs = _by_group(st, x, longest)
    y = torch.bmm(xs, w)[group, place]
    if case["quantized"]:
        y = y * st["scale"][:, None] * st["weight_scale"][group]
    if case["bias"]:
        y = y + st["bias"].detach().float()[group]
    out = [y.to(t)]
    if case["train"]:
        d = _by_group(st, st["d_out"], longest)
        out += [torch.bmm(d, w.transpose(1, 2))[group, place].to(t), torch.bmm(xs.transpose(1, 2), d).to(t)]
        if case["bias"]:
            out.append(d.sum(1).to(t))
    return out


def _noise(step, seed, blocks):
    """16 + 16 bits for every value: a finaliser of a 32-bit hash over its position, keyed by seed and step."""
    low = 0xFFFFFFFF

    def mixed(v):
        v = ((v ^ (v >> 16)) * 0x85EBCA6B) & low
        v = ((v ^ (v >> 13)) * 0xC2B2AE35) & low
        return v ^ (v >> 16)

    key = mixed((step * 0x9E3779B1 + seed) & low)
    place = torch.arange(blocks * BLOCK, device=DEVICE)
    bits = mixed(mixed((place & low) ^ key) ^ (place >> 32)).view(blocks, BLOCK)
    return (bits & 0xFFFF).float() * 2.0 ** -16, (bits >> 16).float() * 2.0 ** -16


def _in_e4m3(values, noise, floor):
    """Blocks of values as e4m3 and a scale, rounded up or down by chance in proportion to the distance."""
    most = values.abs().amax(1, keepdim=True).clamp_min(1e-30)
    y = values * (most.reciprocal() * E4M3_MOST)
    size = y.abs()
    power = ((size.view(torch.int32) >> 23) - 127).clamp_min(-6) - 3            # of the step at that value
    step, per_step = ((power + 127) << 23).view(torch.float32), ((127 - power) << 23).view(torch.float32)
    size = (torch.floor(size * per_step + noise) * step).clamp_max(E4M3_MOST)
    if floor:
        size = torch.where(y > 0, size.clamp_min(2.0 ** -9), size)
    return torch.copysign(size, y).to(torch.float8_e4m3fn), (most * (1.0 / E4M3_MOST))[:, 0]


def _plain_step(st):
    case, f = st["case"], st["flat"]
    st["step"] += 1
    bc1, bc2 = (-torch.expm1(st["step"].double() * math.log(b)) for b in (BETA1, BETA2))
    g, p = f["grad"].float().view(-1, BLOCK), f["param"].view(-1, BLOCK)
    if case["bits"] == 8:
        m = f["exp_avg"].float().view(-1, BLOCK) * f["exp_avg_scale"][:, None]
        r = f["exp_avg_sq"].float().view(-1, BLOCK) * f["exp_avg_sq_scale"][:, None]
        v = r * r
    else:
        m, v = f["exp_avg"].view(-1, BLOCK), f["exp_avg_sq"].view(-1, BLOCK)
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + (g * g) * (1 - BETA2)
    r = torch.sqrt(v)
    p.mul_(1 - LR * DECAY).sub_(m / (r * (1 / torch.sqrt(bc2)).float() + EPS) * (LR / bc1).float())
    if case["bits"] == 8:
        for k, x, u, floor in (("exp_avg", m, 0, False), ("exp_avg_sq", r, 1, True)):
            q, scale = _in_e4m3(x, _noise(st["step"], st["seed"], len(x))[u], floor)
            f[k].copy_(q.view(-1))
            f[k + "_scale"].copy_(scale)
    else:
        f["exp_avg"].copy_(m.view(-1))
        f["exp_avg_sq"].copy_(v.view(-1))
    if case["copies"]:
        f["copy"].copy_(f["param"])
    return _step_outputs(st)


def _step_outputs(st):
    f = st["flat"]
    return {k: f[k] for k in f if k != "grad"} | {"step": st["step"]}


# ---- one pass ---------------------------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if not own:
        return {"norm": _plain_norm, "group": _plain_group, "step": _plain_step}[case["kind"]](state)
    import sparseconvnet_b200 as scn
    st = state
    if case["kind"] == "norm":
        if case["quantized"]:
            return list(scn.rms_norm_quantized(st["x"], st["weight"], residual=st["residual"], eps=NORM_EPS))
        made = scn.rms_norm(st["x"], st["weight"], residual=st["residual"], eps=NORM_EPS)
        out = list(made) if case["residual"] else [made]
        if case["train"]:
            out += torch.autograd.grad(out, [st["x"], st["weight"]], [st["d_out"], st["d_sum"]][:len(out)])
        return out
    if case["kind"] == "group":
        if case["quantized"]:
            return [scn.grouped_product_quantized(st["x"], st["scale"], st["weight"], st["weight_scale"], st["offsets"],
                                                  st["bias"], out_dtype=TYPES[case["type"]])]
        out = [scn.grouped_product(st["x"], st["weight"], st["offsets"], st["bias"])]
        if case["train"]:
            leaves = [t for t in (st["x"], st["weight"], st["bias"]) if t is not None]
            out += torch.autograd.grad(out, leaves, [st["d_out"]])
        return out
    t = st["lists"]
    scn.adamw_step(t["param"], t["grad"], t["exp_avg"], t["exp_avg_sq"], st["step"], lr=LR, betas=(BETA1, BETA2), eps=EPS,
                   weight_decay=DECAY, exp_avg_scales=t.get("exp_avg_scale"), exp_avg_sq_scales=t.get("exp_avg_sq_scale"),
                   seed=st["seed"], copies=t.get("copy"))
    return _step_outputs(st)


def work(case):
    if case["kind"] == "norm":
        values, b = case["rows"] * case["planes"], SIZE[case["type"]]
        moved = values * b * (3 if case["residual"] else 1) + values * (1 if case["quantized"] else b)
        if case["train"]:
            moved += values * b * (3 if case["residual"] else 2)
        return {"bytes": float(moved + 4 * case["planes"] + (4 * case["rows"] if case["quantized"] else 0)),
                "flops": float(values * (14 if case["train"] else 5))}
    if case["kind"] == "group":
        b = 1 if case["quantized"] else SIZE[case["type"]]
        weights = min(case["groups"], case["rows"]) * case["nin"] * case["nout"]
        moved = case["rows"] * (case["nin"] * b + case["nout"] * SIZE[case["type"]]) + weights * b
        if case["train"]:
            moved += case["rows"] * (case["nin"] + case["nout"]) * b + case["groups"] * case["nin"] * case["nout"] * b
        return {"bytes": float(moved), "flops": 2.0 * case["rows"] * case["nin"] * case["nout"] * (3 if case["train"] else 1)}
    values = float(sum(_tensor_sizes(case)))
    each = SIZE[case["grads"]] + 8 + (4 + 16.0 / BLOCK if case["bits"] == 8 else 16) + (2 if case["copies"] else 0)
    return {"bytes": values * each, "flops": values * 15}


# ---- in 64 bits, from the definitions -----------------------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "norm":
        x = st["x"].detach()
        s = x.double()
        if case["residual"]:
            s = (s + st["residual"].double()).to(x.dtype).double()
        root = (s.square().sum(1) / case["planes"] + NORM_EPS).sqrt()[:, None]
        w = st["weight"].detach().double()
        y = s / root * w
        if case["quantized"]:
            most = y.abs().max(1).values
            out = [y / most[:, None] * E4M3_MOST, most / E4M3_MOST]
        else:
            out = [y]
        if case["residual"]:
            out.append(s)
        if case["train"]:
            d = st["d_out"].double()
            along = (d * w * s).sum(1)[:, None] / case["planes"]
            dx = d * w / root - s * along / root ** 3
            if case["residual"]:
                dx = dx + st["d_sum"].double()
            out += [dx, torch.einsum("nc,nc->c", d, s / root)]
        return out
    if case["kind"] == "group":
        edges, x, w = st["offsets"].tolist(), st["x"].detach().double(), st["weight"].detach().double()
        if case["quantized"]:
            x = x * st["scale"].double()[:, None]
            w = (w * st["weight_scale"].double()[:, :, None]).mT
        y = x.new_zeros(case["rows"], case["nout"])
        dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), w.new_zeros(case["groups"], case["nout"])
        for i, (a, b) in enumerate(zip(edges, edges[1:])):
            y[a:b] = x[a:b] @ w[i]
            if case["bias"]:
                y[a:b] += st["bias"][i].detach().double()
            if case["train"]:
                d = st["d_out"][a:b].double()
                dx[a:b], dw[i], db[i] = d @ w[i].T, x[a:b].T @ d, d.sum(0)
        return [y] + ([dx, dw] if case["train"] else []) + ([db] if case["train"] and case["bias"] else [])
    f, t = st["flat"], STEPS_DONE + 1
    wide = lambda k: f[k].double() * f[k + "_scale"].double().repeat_interleave(BLOCK) if case["bits"] == 8 else f[k].double()  # noqa: E731
    g, m, v = f["grad"].double(), wide("exp_avg"), wide("exp_avg_sq")
    if case["bits"] == 8:
        v = v.square()
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g.square()
    p = f["param"].double()
    p = p - LR * DECAY * p - LR * (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + EPS)
    out = {"param": p, "step": torch.tensor([t], device=DEVICE)}
    if case["bits"] == 8:  # codes are rounded by chance: they have no value of their own, their scales have
        scale = lambda x: x.view(-1, BLOCK).abs().amax(1).clamp_min(1e-30) / E4M3_MOST  # noqa: E731
        out.update(exp_avg=None, exp_avg_scale=scale(m), exp_avg_sq=None, exp_avg_sq_scale=scale(v.sqrt()))
    else:
        out.update(exp_avg=m, exp_avg_sq=v)
    if case["copies"]:
        out["copy"] = p
    return out
