"""Measured cases of the operators that train and look up what a model has learned.

* ``lookup``  rows of an embedding table times a scale (``landmark_b200.embedding.embedding``): an appearance code per ray
              or per sample, a token's row;
* ``grad``    the gradient of that table (``landmark_b200.embedding.embedding_backward``): the output's rows summed by
              index, every row of the table written;
* ``adamw``   one AdamW step over many tensors at once (``landmark_b200.optim.AdamWTensors``), with states in 32 bits or in
              blocks of 8-bit codes.

``run`` computes each either in elementary torch operations (``own`` false) or through the package.
"""
import math
import random

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}
BLOCK = 256  # values that share a scale in the 8-bit states
TOP = 448.0  # largest e4m3 value
MASK = 0xFFFFFFFF


# -- cases ---------------------------------------------------------------------------------------------------------------


def _rows(name, op, tokens, rows, dim, dtype, spread, distinct=0, scale=1.0, masked=0.0, index="int64", out="", accumulate=False):
    """``spread``: ``runs`` (every sample of a ray has its ray's code, ``distinct`` codes in all), ``zipf`` or ``uniform``.
    ``masked``: share of negative indices.  ``out``: type of the gradient, the table's if empty."""
    c = {"op": op, "tokens": tokens, "rows": rows, "dim": dim, "dtype": dtype, "spread": spread, "distinct": distinct, "scale": scale,
         "masked": masked, "index": index}
    if op == "grad":
        c.update({"out": out or dtype, "accumulate": accumulate})
    if name:
        c["name"] = name
    return c


def _adamw(name, layout, bits, param="fp32", grad="fp32", master=False, scale=1, tensors=0, values=0, packed=False, step=1, lr=1e-3,
           beta1=0.9, beta2=0.999, decay=0.01):
    """``layout``: ``field`` (planes and lines of the city grid over ``scale``), ``network`` (basis, colour network and
    appearance table) or ``mixed`` (``tensors`` tensors of about ``values`` values together, sizes from 1 up).  ``packed``: the tensors lie
    in one buffer without a gap, whatever alignment that gives them."""
    c = {"op": "adamw", "layout": layout, "bits": bits, "param": param, "grad": grad, "master": master, "scale": scale,
         "tensors": tensors, "values": values, "packed": packed, "step": step, "lr": lr, "beta1": beta1, "beta2": beta2, "decay": decay}
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # the latent of one view
        _rows("lookup_one_code", "lookup", 1, 11500, 48, "fp32", "uniform"),
        # a row for every appearance sample of a few render chunks, some samples masked
        _rows("lookup_samples", "lookup", 1500007, 11500, 48, "fp32", "runs", distinct=600, masked=0.05),
        # token rows of a large vocabulary, scaled by the root of the width
        _rows("lookup_tokens_bf16", "lookup", 32768, 131072, 2048, "bf16", "zipf", scale=math.sqrt(2048.0), index="int32"),
        # a few rays of one new photograph: every sample has the same code
        _rows("grad_one_code", "grad", 333, 11500, 48, "fp32", "runs", distinct=1),
        # the samples of a training batch of rays: long runs, few codes
        _rows("grad_samples", "grad", 1500007, 11500, 48, "fp32", "runs", distinct=600, masked=0.05),
        # a batch of tokens, gradient in 32 bits added to that of the micro-batches before
        _rows("grad_tokens_bf16", "grad", 16384, 131072, 2048, "bf16", "zipf", scale=math.sqrt(2048.0), out="fp32", accumulate=True),
        # odd vocabulary and width in half precision
        _rows("grad_odd_fp16", "grad", 5003, 50021, 771, "fp16", "zipf", masked=0.1, index="int32"),
        # appearance table, basis and network of one model
        _adamw("adamw_network", "network", 32, step=17, beta2=0.99, decay=0.0),
        # every plane and line of the city block, states in 32 bits ...
        _adamw("adamw_field", "field", 32, step=1000, lr=2e-2, beta2=0.99, decay=0.0),
        # ... and in 8
        _adamw("adamw_field_8bit", "field", 8, step=1000, lr=2e-2, beta2=0.99, decay=0.0),
        # some hundred 16-bit weights with 32-bit copies
        _adamw("adamw_mixed_bf16", "mixed", 32, param="bf16", grad="bf16", master=True, tensors=300, values=60000000, step=1),
        # the same kind with 8-bit states, tensors of any size packed without gaps
        _adamw("adamw_packed_8bit", "mixed", 8, param="bf16", grad="bf16", master=True, tensors=90, values=9000001, packed=True, step=3),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["lookup", "grad", "grad", "adamw", "adamw"])
    if op == "adamw":
        layout = rng.choice(["field", "network", "mixed", "mixed"])
        bits = rng.choice([8, 32])
        param = rng.choice(["fp32", "bf16", "bf16", "fp16"]) if layout == "mixed" else "fp32"
        grad = rng.choice([param, param, "fp32"]) if param != "fp32" else rng.choice(["fp32", "fp32", "bf16", "fp16"])
        tensors = _log(rng, 1, 400)
        return _adamw("", layout, bits, param, grad, param != "fp32" and rng.random() < 0.7, scale=rng.choice([2, 4, 8]) if layout == "field" else 1,
                      tensors=tensors if layout == "mixed" else 0, values=max(tensors, _log(rng, 1000, 80000000)) if layout == "mixed" else 0,
                      packed=rng.random() < 0.3, step=_log(rng, 1, 100000), lr=10 ** rng.uniform(-4, -2), beta2=rng.choice([0.95, 0.99, 0.999]),
                      decay=rng.choice([0.0, 0.01, 0.1]))
    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    if rng.random() < 0.5:
        tokens, rows, dim, spread = _log(rng, 1, 1500000), 11500, 48, "runs"
    else:
        tokens, rows, dim, spread = _log(rng, 1, 20000), _log(rng, 100, 131072), _log(rng, 8, 2048), rng.choice(["zipf", "zipf", "uniform"])
        if rng.random() < 0.5:
            dim = max(8, dim // 64 * 64)
    return _rows("", op, tokens, rows, dim, dtype, spread, distinct=_log(rng, 1, 2000) if spread == "runs" else 0,
                 scale=rng.choice([1.0, math.sqrt(dim), 0.37]), masked=rng.choice([0.0, 0.0, 0.05, 0.3]), index=rng.choice(["int64", "int32"]),
                 out=rng.choice([dtype, "fp32"]), accumulate=rng.random() < 0.3)


def _sizes(case):
    """Numbers of values of the tensors of an optimiser step."""
    if case["layout"] == "network":
        return [27 * 144, 128 * 198, 128, 128 * 128, 128, 3 * 128, 3, 11500 * 48]
    if case["layout"] == "field":
        x, z = 2048 // case["scale"], 256 // case["scale"]
        return [n for c in (16, 48) for n in (c * x * x, c * x * z, c * x * z, c * z, c * x, c * x)]
    rng = random.Random(case["tensors"] * 1000003 + case["values"])
    share = [math.exp(rng.uniform(0.0, math.log(1000.0))) for _ in range(case["tensors"])]
    total = sum(share)
    return [max(1, int(case["values"] * s / total)) for s in share]


def _starts(case):
    """Where each tensor begins in the buffer of them all, and the buffer's size."""
    at, starts = 0, []
    for n in _sizes(case):
        starts.append(at)
        at += n if case["packed"] else -(-n // 64) * 64
    return starts, at


# -- inputs --------------------------------------------------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _indices(case, gen):
    t, v = case["tokens"], case["rows"]
    if case["spread"] == "runs":
        codes = torch.randint(0, v, (case["distinct"],), generator=gen, device=DEVICE)
        ray = torch.cumsum((torch.rand(t, generator=gen, device=DEVICE) < 1.0 / 24).long(), 0)
        of_ray = codes[torch.randint(0, case["distinct"], (t + 1,), generator=gen, device=DEVICE)]
        idx = of_ray[ray]
    else:
        u = torch.rand(t, generator=gen, device=DEVICE, dtype=torch.float64)
        idx = (v * (u * u if case["spread"] == "zipf" else u)).long().clamp_(max=v - 1)
        idx = (idx * 7919) % v if math.gcd(7919, v) == 1 else idx  # frequent rows are not neighbours
    if case["masked"]:
        idx = torch.where(torch.rand(t, generator=gen, device=DEVICE) < case["masked"], torch.full_like(idx, -1), idx)
    return idx.to(torch.int32) if case["index"] == "int32" else idx


def _randn(n, gen, scale, dtype):
    return torch.randn(n, generator=gen, device=DEVICE).mul_(scale).to(dtype)


def _to_codes(x, sizes, starts):
    """Nearest 8-bit codes and block scales of a buffer of values: a state that earlier steps have left."""
    codes = torch.zeros(x.numel(), device=DEVICE, dtype=torch.float8_e4m3fn)
    scales = []
    for n, at in zip(sizes, starts):
        b = torch.nn.functional.pad(x[at:at + n], (0, -n % BLOCK)).view(-1, BLOCK)
        s = b.abs().amax(1) / TOP
        codes[at:at + n] = (b / s.clamp(min=1e-38)[:, None]).clamp(-TOP, TOP).view(-1)[:n].to(torch.float8_e4m3fn)
        scales.append(s)
    return codes, torch.cat(scales)


def prepare(case, seed):
    gen = _generator(seed)
    if case["op"] == "lookup":
        return {"case": case, "indices": _indices(case, gen),
                "weight": _randn((case["rows"], case["dim"]), gen, 1.0 if case["spread"] == "runs" else 0.02, DTYPES[case["dtype"]])}
    if case["op"] == "grad":
        s = {"case": case, "indices": _indices(case, gen), "grad": _randn((case["tokens"], case["dim"]), gen, 1e-2, DTYPES[case["dtype"]])}
        if case["accumulate"]:
            s["into"] = _randn((case["rows"], case["dim"]), gen, 1e-2, DTYPES[case["out"]])
        return s
    sizes = _sizes(case)
    starts, total = _starts(case)
    master = _randn(total, gen, 0.1, torch.float32)
    g = _randn(total, gen, 1e-3, torch.float32)
    g *= torch.exp(_randn(total, gen, 1.0, torch.float32))  # gradients of a field differ by orders of magnitude
    m = torch.zeros(total, device=DEVICE) if case["step"] == 1 else g * _randn(total, gen, 0.3, torch.float32)
    v = torch.zeros(total, device=DEVICE) if case["step"] == 1 else g * g * (0.1 + torch.rand(total, generator=gen, device=DEVICE))
    s = {"case": case, "step": case["step"], "seed": seed & 0xFFFF, "p": master if case["param"] == "fp32" else master.to(DTYPES[case["param"]]),
         "g": g.to(DTYPES[case["grad"]])}
    if case["master"]:
        s["master"] = master
    if case["bits"] == 8:
        s["m"], s["ms"] = _to_codes(m, sizes, starts)
        s["v"], s["vs"] = _to_codes(v.sqrt(), sizes, starts)
    else:
        s["m"], s["v"] = m, v
    cut = lambda x: [x[at:at + n] for n, at in zip(sizes, starts)]  # noqa: E731
    s["views"] = {k: cut(s[k]) for k in ("p", "g", "m", "v", "master") if k in s}
    if case["bits"] == 8:
        blocks = [-(-n // BLOCK) for n in sizes]
        s["views"].update({k: list(torch.split(s[k], blocks)) for k in ("ms", "vs")})
    return s


# -- the calls of the package ----------------------------------------------------------------------------------------------


def _run_own(s):
    from landmark_b200.embedding import embedding, embedding_backward
    from landmark_b200.optim import AdamWTensors

    c = s["case"]
    if c["op"] == "lookup":
        return embedding(s["indices"], s["weight"], scale=c["scale"])
    if c["op"] == "grad":
        if c["accumulate"]:
            return embedding_backward(s["grad"], s["indices"], c["rows"], scale=c["scale"], out=s["into"], accumulate=True)
        return embedding_backward(s["grad"], s["indices"], c["rows"], scale=c["scale"], dtype=DTYPES[c["out"]])
    w = s["views"]
    if "tensors" not in s:  # a trainer's parameters and states, checked when it starts
        s["tensors"] = AdamWTensors(w["p"], w["m"], w["v"], w.get("ms"), w.get("vs"), w.get("master"))
    s["tensors"].step(w["g"], step=s["step"], lr=c["lr"], betas=(c["beta1"], c["beta2"]), eps=1e-8, weight_decay=c["decay"], seed=s["seed"])


# -- plain forms -----------------------------------------------------------------------------------------------------------


def _hash(i, seed):
    """32 well mixed bits of the 32-bit numbers ``i`` (an int64 tensor or an int) and a seed."""
    x = (i * 0x9E3779B9 + seed) & MASK
    x = x ^ (x >> 16)
    x = (x * 0x6A09E667) & MASK
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & MASK
    return x ^ (x >> 16)


def _floor_e4m3(y):
    """Largest e4m3 value that is not above ``y`` in [0, 448], and the distance to the next one."""
    bits = y.view(torch.int32)
    low = torch.where(y < 2.0 ** -6, torch.floor(y * 512) / 512, (bits & ~0xFFFFF).view(torch.float32))
    return low, (bits & 0x7F800000).view(torch.float32).clamp(min=2.0 ** -6) / 8


def _blocks(x):
    return torch.nn.functional.pad(x, (0, -x.numel() % BLOCK)).view(-1, BLOCK)


def _encode(x, unit, squared, codes, scales):
    """``x`` into 8-bit codes and block scales, rounded up with the probability that keeps the mean of ``x`` (``squared``: of
    its square, and then never to zero).  ``unit``: a uniform number in (0, 1) for each value."""
    b = _blocks(x)
    top = torch.where(torch.isfinite(b), b.abs(), torch.zeros_like(b)).amax(1)
    top = torch.where(top < 1e-30, torch.zeros_like(top), top)
    y = (b.abs() * torch.where(top > 0, TOP / top, top)[:, None]).clamp(max=TOP)
    low, step = _floor_e4m3(torch.nan_to_num(y))
    u = _blocks(unit)
    if squared:
        up = u * (2 * low + step) * step < (y - low) * (y + low)
    else:
        up = u * step < y - low
    c = low + torch.where(up, step, torch.zeros_like(step))
    if squared:
        c = torch.where((y > 0) & (c == 0), torch.full_like(c, 2.0 ** -9), c)
    c = torch.where(torch.isfinite(b), torch.copysign(c, b), torch.full_like(c, float("nan")))
    codes.copy_(c.view(-1)[:x.numel()].to(torch.float8_e4m3fn))
    scales.copy_(top / TOP)


def _decode(codes, scales):
    return codes.float() * scales.repeat_interleave(BLOCK)[:codes.numel()]


def _adamw_plain(s):
    c, w, t = s["case"], s["views"], s["step"]
    b1, b2, lr = c["beta1"], c["beta2"], c["lr"]
    c1, c2 = 1 - b1 ** t, math.sqrt(1 - b2 ** t)
    seed = _hash(t, s["seed"])
    for k in range(len(w["p"])):
        p, g, eight = w["p"][k], w["g"][k].float(), c["bits"] == 8
        m = _decode(w["m"][k], w["ms"][k]) if eight else w["m"][k]
        v = _decode(w["v"][k], w["vs"][k]).square() if eight else w["v"][k]
        m = b1 * m + (1 - b1) * g
        v = b2 * v + (1 - b2) * g * g
        x = w["master"][k] if c["master"] else p.float()
        x = x * (1 - lr * c["decay"]) - (lr / c1) * (m / (torch.sqrt(v) / c2 + 1e-8))
        p.copy_(x)
        if c["master"]:
            w["master"][k].copy_(x)
        if eight:
            h = _hash(torch.arange(p.numel(), device=p.device), _hash(k, seed))
            _encode(m, ((h & 0xFFFF).float() + 0.5) / 65536, False, w["m"][k], w["ms"][k])
            _encode(torch.sqrt(v), ((h >> 16).float() + 0.5) / 65536, True, w["v"][k], w["vs"][k])
        else:
            w["m"][k].copy_(m)
            w["v"][k].copy_(v)


def _run_plain(s):
    c = s["case"]
    if c["op"] == "lookup":
        idx = s["indices"].long()
        rows = s["weight"][idx.clamp(min=0)].float() * c["scale"]
        return torch.where((idx >= 0)[:, None], rows, torch.zeros_like(rows)).to(s["weight"].dtype)
    if c["op"] == "grad":
        idx = s["indices"].long()
        # long sums of both signs: in 64 bits; the masked ones go to a row of their own
        total = torch.zeros((c["rows"] + 1, c["dim"]), dtype=torch.float64, device=DEVICE)
        total.index_add_(0, torch.where(idx < 0, torch.full_like(idx, c["rows"]), idx), s["grad"].double())
        total = total[:-1] * c["scale"]
        if c["accumulate"]:
            return s["into"].copy_(total + s["into"])
        return total.to(DTYPES[c["out"]])
    _adamw_plain(s)


def run(state):
    out = _run_own(state) if own else _run_plain(state)
    if state["case"]["op"] != "adamw":
        return out
    state["step"] += 1
    return {k: state[k] for k in ("p", "m", "v", "ms", "vs", "master") if k in state}


# -- 64 bits ---------------------------------------------------------------------------------------------------------------


def _exact_codes(x, unit, squared):
    """(values of the codes, scales) from a table of the e4m3 values."""
    table = torch.tensor([k * 2.0 ** -9 for k in range(8)] + [(1 + k / 8) * 2.0 ** e for e in range(-6, 9) for k in range(8)][:-1],
                         dtype=torch.float64, device=DEVICE)
    b = torch.nn.functional.pad(x, (0, -x.numel() % BLOCK)).view(-1, BLOCK)
    scale = b.abs().amax(1) / TOP
    scale[scale < 1e-30 / TOP] = 0
    y = (b.abs() / torch.where(scale > 0, scale, torch.ones_like(scale))[:, None]).view(-1)[:x.numel()].clamp(max=TOP)
    y = y * (scale > 0).repeat_interleave(BLOCK)[:x.numel()]
    k = torch.searchsorted(table, y, right=True) - 1
    lo, hi = table[k], table[(k + 1).clamp(max=table.numel() - 1)]
    if squared:
        up = unit * (hi ** 2 - lo ** 2) < y ** 2 - lo ** 2
    else:
        up = unit * (hi - lo) < y - lo
    z = torch.where(up, hi, lo)
    if squared:
        z = torch.where((y > 0) & (z == 0), torch.full_like(z, 2.0 ** -9), z)
    return torch.sign(x) * z, scale


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "lookup":
        w = torch.cat([s["weight"].double() * case["scale"], torch.zeros((1, case["dim"]), dtype=torch.float64, device=DEVICE)])
        return w.index_select(0, s["indices"].long().remainder(case["rows"] + 1))  # -1: the last row
    if case["op"] == "grad":
        order = torch.argsort(s["indices"].long(), stable=True)
        key = s["indices"].long()[order]
        upto = torch.cumsum(torch.cat([torch.zeros((1, case["dim"]), dtype=torch.float64, device=DEVICE), s["grad"][order].double()]), 0)
        edge = torch.searchsorted(key, torch.arange(case["rows"] + 1, device=DEVICE))
        total = (upto[edge[1:]] - upto[edge[:-1]]) * case["scale"]
        return total + s["into"].double() if case["accumulate"] else total
    t, b1, b2 = case["step"], case["beta1"], case["beta2"]
    outs = {k: s[k].double() for k in ("p", "m", "v", "ms", "vs", "master") if k in s}
    first = _hash(t, s["seed"])
    at8 = 0
    for k, (n, at) in enumerate(zip(_sizes(case), _starts(case)[0])):
        cut = slice(at, at + n)
        g = s["g"][cut].double()
        m, v = outs["m"][cut], outs["v"][cut]
        if case["bits"] == 8:
            cut8 = slice(at8, at8 + -(-n // BLOCK))
            at8 = cut8.stop
            m = m * outs["ms"][cut8].repeat_interleave(BLOCK)[:n]
            v = (v * outs["vs"][cut8].repeat_interleave(BLOCK)[:n]) ** 2
        m = m + (1 - b1) * (g - m)
        v = v + (1 - b2) * (g * g - v)
        x = outs["master" if case["master"] else "p"][cut]
        x = x - case["lr"] * (case["decay"] * x + (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + 1e-8))
        for key in ("p", "master"):
            if key in outs:
                outs[key][cut] = x
        if case["bits"] == 8:
            h = _hash(torch.arange(n, device=DEVICE), _hash(k, first))
            m, outs["ms"][cut8] = _exact_codes(m, ((h % 65536).double() + 0.5) / 65536, False)
            v, outs["vs"][cut8] = _exact_codes(torch.sqrt(v), ((h // 65536).double() + 0.5) / 65536, True)
        outs["m"][cut], outs["v"][cut] = m, v
    return outs


# -- what a pass cannot do without -----------------------------------------------------------------------------------------


def _distinct(case):
    """Rows that the indices name, on average."""
    t, v = case["tokens"] * (1 - case["masked"]), case["rows"]
    if case["spread"] == "runs":
        return min(case["distinct"], t)
    if case["spread"] == "uniform":
        return v * -math.expm1(t * math.log1p(-1.0 / v)) if v > 1 else 1.0
    n, total = 512, 0.0  # row r of `v` comes with probability sqrt((r + 1) / v) - sqrt(r / v)
    for k in range(n):
        lo, hi = (k / n) ** 2 * v, ((k + 1) / n) ** 2 * v
        p = (1.0 / n) / max(hi - lo, 1.0)
        total += min(hi - lo, 1.0) if hi - lo < 1 else (hi - lo) * -math.expm1(t * math.log1p(-min(p, 1 - 1e-9)))
    return min(total, t, v)


def work(case):
    if case["op"] == "adamw":
        n = sum(_sizes(case))
        per = BYTES[case["param"]] * (1 if case["master"] else 2) + (8 if case["master"] else 0) + BYTES[case["grad"]]
        per += 16 if case["bits"] == 32 else 4 + 16.0 / BLOCK
        return {"bytes": n * per, "flops": 15.0 * n}
    rows, e = case["tokens"] * case["dim"], BYTES[case["dtype"]]
    index = case["tokens"] * (4 if case["index"] == "int32" else 8)
    if case["op"] == "lookup":
        return {"bytes": rows * e + index + _distinct(case) * case["dim"] * e, "flops": float(rows)}
    # a masked row is not read; with accumulate only the rows that are named change
    table = _distinct(case) * 2 if case["accumulate"] else case["rows"]
    return {"bytes": rows * e * (1 - case["masked"]) + index + table * case["dim"] * BYTES[case["out"]], "flops": rows * (1 - case["masked"])}
