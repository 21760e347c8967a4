"""AdamW steps against the formula in 64 bits.

With u = 2^-24, each rounded operation of the step is off by at most u of its result:
  m = b1 m + b1c g      3 u |b1 m| + 3 u |b1c g|  (coefficient, product, sum), rounded up to 4 u each
  v                     all terms positive: 5 u |v|
  update = rate * (m / (sqrt(v) / c2 + eps)): the error of m over the same denominator, and of itself 2.5 u for v's error under
                        the root, 1 for the root, 2 for 1 / c2 and its product, 1 for the sum, 2 for a reciprocal within one unit
                        of the last place, 1 for its product with m, 2 for rate and its product: 11.5 u, rounded up to 12
  p = keep p - update   3 u |keep p| + u |p|"""
import copy
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BLOCK = 256
TOP = 448.0


def reference(x, g, m, v, step, lr, betas, eps, decay):
    """(p, m, v) and how far each may be off, from 64-bit inputs."""
    b1, b2 = betas
    m2, v2 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    m_tol, v_tol = 4 * U * (b1 * m.abs() + (1 - b1) * g.abs()), 5 * U * v2
    rate, c2 = lr / (1 - b1 ** step), math.sqrt(1 - b2 ** step)
    denominator = torch.sqrt(v2) / c2 + eps
    update = rate * m2 / denominator
    p = x * (1 - lr * decay) - update
    return (p, m2, v2), (rate * m_tol / denominator + 12 * U * update.abs() + 3 * U * x.abs() + U * p.abs(), m_tol, v_tol)


def tensors(sizes, dtype, grad, seed=0, packed=False):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    starts, at = [], 0
    for n in sizes:
        starts.append(at)
        at += n if packed else -(-n // 64) * 64
    flat = [torch.randn(at, generator=gen, device="cuda") * s for s in (0.1, 1e-3, 1e-3)] + [torch.rand(at, generator=gen, device="cuda") * 1e-6]
    flat[1] *= torch.exp(torch.randn(at, generator=gen, device="cuda"))
    cut = [[f[a:a + n] for n, a in zip(sizes, starts)] for f in flat]
    p = flat[0].to(dtype)
    g = flat[1].to(grad)
    return [p[a:a + n] for n, a in zip(sizes, starts)], [g[a:a + n] for n, a in zip(sizes, starts)], cut[2], cut[3], cut[0]


SIZES = [1, 2, 3, 4, 5, 127, 255, 256, 257, 1000, 4095, 4096, 4097, 70001]
MIXES = [(torch.float32, torch.float32, False), (torch.float32, torch.bfloat16, False), (torch.bfloat16, torch.bfloat16, True),
         (torch.bfloat16, torch.float32, True), (torch.float16, torch.float16, True), (torch.bfloat16, torch.bfloat16, False),
         (torch.float16, torch.float32, False)]


@pytest.mark.parametrize("dtype,grad,master", MIXES)
@pytest.mark.parametrize("packed", [False, True])
def test_step_32bit(dtype, grad, master, packed):
    from landmark_b200.optim import adamw_step

    for step, betas, decay in ((1, (0.9, 0.999), 0.1), (1000, (0.9, 0.99), 0.0)):
        p, g, m, v, x = tensors(SIZES, dtype, grad, packed=packed)
        if not master:
            x = [t.float() for t in p]
        want = [reference(a.double(), b.double(), c.double(), d.double(), step, 1e-2, betas, 1e-8, decay) for a, b, c, d in zip(x, g, m, v)]
        adamw_step(p, g, m, v, step=step, lr=1e-2, betas=betas, weight_decay=decay, masters=x if master else None)
        for k, ((rp, rm, rv), (tp, tm, tv)) in enumerate(want):
            assert bool(((m[k].double() - rm).abs() <= tm).all()) and bool(((v[k].double() - rv).abs() <= tv).all()), SIZES[k]
            if master:
                assert bool(((x[k].double() - rp).abs() <= tp).all()), SIZES[k]
                assert torch.equal(p[k], x[k].to(dtype))
            else:
                off = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2 * (rp.abs() + tp) + (2.0 ** -25 if dtype == torch.float16 else 0)
                assert bool(((p[k].double() - rp).abs() <= tp + off).all()), SIZES[k]


# -- 8-bit states: the same separately rounded fp32 operations in torch ------------------------------------------------------


def hash32(i, seed):
    mask = 0xFFFFFFFF
    x = (i * 0x9E3779B9 + seed) & mask
    x = x ^ (x >> 16)
    x = (x * 0x6A09E667) & mask
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & mask
    return x ^ (x >> 16)


def encode(x, unit, squared):
    pad = -x.numel() % BLOCK
    b, u = torch.nn.functional.pad(x, (0, pad)).view(-1, BLOCK), torch.nn.functional.pad(unit, (0, pad)).view(-1, BLOCK)
    fine = torch.isfinite(b)
    top = torch.where(fine, b.abs(), torch.zeros_like(b)).amax(1)
    top = torch.where(top < 1e-30, torch.zeros_like(top), top)
    inv = torch.where(top > 0, top.reciprocal() * TOP, torch.zeros_like(top))
    y = torch.where(fine, b.abs() * inv[:, None], torch.zeros_like(b)).clamp(max=TOP)
    low = torch.where(y < 2.0 ** -6, torch.floor(y * 512) / 512, (y.view(torch.int32) & ~0xFFFFF).view(torch.float32))
    step = (y.view(torch.int32) & 0x7F800000).view(torch.float32).clamp(min=2.0 ** -6) / 8
    up = u * (2 * low + step) * step < (y - low) * (y + low) if squared else u * step < y - low
    c = torch.where(up, low + step, low)
    if squared:
        c = torch.where((y > 0) & (c == 0), torch.full_like(c, 2.0 ** -9), c)
    c = torch.where(fine, torch.copysign(c, b), torch.full_like(c, float("nan")))
    return c.view(-1)[:x.numel()], top * (1 / TOP)


def random_states(sizes, seed=3):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    codes = [[(torch.randn(n, generator=gen, device="cuda") * 60).clamp(-448, 448).to(torch.float8_e4m3fn) for n in sizes],
             [(torch.rand(n, generator=gen, device="cuda") * 448).to(torch.float8_e4m3fn) for n in sizes]]
    scales = [[torch.rand(-(-n // BLOCK), generator=gen, device="cuda") * s for n in sizes] for s in (1e-5, 1e-6)]
    return codes[0], codes[1], scales[0], scales[1]


def bits(t):
    return t.view(torch.uint8)


@pytest.mark.parametrize("dtype,grad,master", MIXES)
@pytest.mark.parametrize("packed", [False, True])
def test_step_8bit(dtype, grad, master, packed):
    from landmark_b200.optim import adamw_step

    step, betas, seed = 37, (0.9, 0.999), 12345
    p, g, _, _, x = tensors(SIZES, dtype, grad, packed=packed)
    if not master:
        x = [t.float() for t in p]
    m, v, ms, vs = random_states(SIZES)
    if packed:  # codes that begin at any byte
        flat = torch.cat([bits(t) for t in m]), torch.cat([bits(t) for t in v])
        m, v = ([f.view(torch.float8_e4m3fn)[a:a + n] for a, n in zip([sum(SIZES[:k]) for k in range(len(SIZES))], SIZES)] for f in flat)
    want = []
    for k, n in enumerate(SIZES):
        wide = lambda s: s.repeat_interleave(BLOCK)[:n]  # noqa: E731
        m32, root = m[k].float() * wide(ms[k]), v[k].float() * wide(vs[k])
        v32, g32 = root * root, g[k].float()
        f32 = lambda c: torch.tensor(c, dtype=torch.float32, device="cuda")  # noqa: E731
        ref = reference(x[k].double(), g32.double(), m32.double(), v32.double(), step, 1e-2, betas, 1e-8, 0.1)
        m32 = f32(betas[0]) * m32 + f32(1 - betas[0]) * g32
        v32 = f32(betas[1]) * v32 + f32(1 - betas[1]) * g32 * g32
        h = hash32(torch.arange(n, device="cuda"), hash32(k, hash32(step, seed)))
        want.append((ref, encode(m32, ((h & 0xFFFF).float() + 0.5) / 65536, False), encode(torch.sqrt(v32), ((h >> 16).float() + 0.5) / 65536, True)))
    adamw_step(p, g, m, v, step=step, lr=1e-2, betas=betas, weight_decay=0.1, exp_avg_scales=ms, exp_avg_sq_scales=vs,
               masters=x if master else None, seed=seed)
    for k, (((rp, _, _), (tp, _, _)), (mc, mscale), (vc, vscale)) in enumerate(want):
        assert torch.equal(ms[k], mscale) and torch.equal(vs[k], vscale), SIZES[k]
        assert torch.equal(m[k].float(), mc) and torch.equal(v[k].float(), vc), SIZES[k]
        if master:
            assert bool(((x[k].double() - rp).abs() <= tp).all()) and torch.equal(p[k], x[k].to(dtype))
        else:
            off = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2 * (rp.abs() + tp) + (2.0 ** -25 if dtype == torch.float16 else 0)
            assert bool(((p[k].double() - rp).abs() <= tp + off).all()), SIZES[k]


def fresh_8bit(n):
    return ([torch.zeros(n, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2)],
            [torch.zeros(-(-n // BLOCK), device="cuda") for _ in range(2)])


def test_8bit_rounding_keeps_the_mean():
    """A step that starts from zero states has m = (1 - b1) g and v = (1 - b2) g^2 exactly; over 1024 seeds the mean of what the codes
    stand for may be off by 6 standard errors of a variable within one code step (standard deviation at most half of it), and by the
    2^-17 that 16 random bits leave of a step."""
    from landmark_b200.optim import adamw_step

    n, seeds = 512, 1024
    g = torch.randn(n, device="cuda") * torch.exp(torch.randn(n, device="cuda"))
    m_sum, v_sum = torch.zeros(n, dtype=torch.float64, device="cuda"), torch.zeros(n, dtype=torch.float64, device="cuda")
    for seed in range(seeds):
        (m, v), (ms, vs) = fresh_8bit(n)
        adamw_step([torch.zeros(n, device="cuda")], [g], [m], [v], step=1, lr=0.0, exp_avg_scales=[ms], exp_avg_sq_scales=[vs], seed=seed)
        m_sum += m.double() * ms.double().repeat_interleave(BLOCK)
        v_sum += (v.double() * vs.double().repeat_interleave(BLOCK)) ** 2
    allowed = 6 * 0.5 / math.sqrt(seeds) + 2.0 ** -17
    for total, exact, scale in ((m_sum, 0.1 * g.double(), ms), (v_sum, 1e-3 * g.double() ** 2, vs)):
        s = scale.double().repeat_interleave(BLOCK)
        y = exact.abs() / s if total is m_sum else exact.sqrt() / s
        width = torch.exp2(torch.floor(torch.log2(y.clamp(2.0 ** -6, 447.9)))) / 8  # one code
        width = width * s if total is m_sum else (2 * y + width) * width * s * s
        assert bool(((total / seeds - exact).abs() <= allowed * width + 1e-6 * exact.abs()).all())


def test_8bit_special_values():
    from landmark_b200.optim import adamw_step

    n = 3 * BLOCK + 5
    g = torch.randn(n, device="cuda") * 1e-3
    g[10], g[BLOCK + 3] = float("nan"), float("inf")
    g[2 * BLOCK:3 * BLOCK] = 0.0
    g[3 * BLOCK] = 1e-12  # beside values a million times as large
    p = torch.randn(n, device="cuda")
    before = p.clone()
    (m, v), (ms, vs) = fresh_8bit(n)
    adamw_step([p], [g], [m], [v], step=1, lr=1e-2, weight_decay=0.0, exp_avg_scales=[ms], exp_avg_sq_scales=[vs])
    bad = torch.zeros(n, dtype=torch.bool, device="cuda")
    bad[10] = bad[BLOCK + 3] = True
    assert torch.equal(p.isfinite(), ~bad) and torch.equal(m.float().isfinite(), ~bad) and torch.equal(v.float().isfinite(), ~bad)
    assert bool(ms.isfinite().all()) and float(ms[2]) == 0 and float(vs[2]) == 0 and torch.equal(p[2 * BLOCK:3 * BLOCK], before[2 * BLOCK:3 * BLOCK])
    assert float(v[3 * BLOCK].float()) == 2.0 ** -9  # never 0 where v is not
    for t in range(2, 30):  # the rest goes on; no value runs away
        g[10] = g[BLOCK + 3] = 1e-3
        adamw_step([p], [g], [m], [v], step=t, lr=1e-2, weight_decay=0.0, exp_avg_scales=[ms], exp_avg_sq_scales=[vs], seed=t)
    assert float((p - before)[~bad].abs().max()) <= 29 * 1e-2 * math.sqrt(10)


def test_many_tensors_and_missing_gradients():
    """More tensors than one launch takes, some without values, some without a gradient."""
    from landmark_b200.optim import AdamWTensors

    sizes = [(7 * k) % 300 for k in range(1001)]
    for eight in (False, True):
        p, g, m, v, _ = tensors(sizes, torch.float32, torch.float32)
        scales = ()
        if eight:
            m, v, *scales = random_states(sizes)
        grads = [None if k % 5 == 0 else t for k, t in enumerate(g)]
        before = [[bits(t.contiguous()).clone() for t in ts] for ts in (p, m, v)]
        one = [[t.clone() for t in ts] for ts in (p, m, v, *scales)]
        AdamWTensors(p, m, v, *scales).step(grads, step=4, lr=1e-3, seed=9)
        for k in range(1001):
            if grads[k] is None:
                assert all(torch.equal(bits(t[k]), b[k]) for t, b in zip((p, m, v), before))
        # in several smaller steps: the same (32 bits) whatever the tensors beside them
        if not eight:
            for lo in range(0, 1001, 143):
                cut = slice(lo, lo + 143)
                AdamWTensors(one[0][cut], one[1][cut], one[2][cut]).step(grads[cut], step=4, lr=1e-3)
            assert all(torch.equal(a, b) for ts, us in zip((p, m, v), one) for a, b in zip(ts, us))


def test_optimiser_follows_the_formula():
    """Ten steps of the class, groups of different rates, a parameter that sometimes has no gradient, against 64 bits; every step adds at
    most the errors above, and an error of p is carried on unchanged."""
    from landmark_b200.optim import AdamW

    torch.manual_seed(0)
    p = [torch.nn.Parameter(torch.randn(n, device="cuda")) for n in ((5, 7), (300,), ())]
    opt = AdamW([{"params": p[:2], "lr": 1e-2}, {"params": p[2:], "betas": (0.8, 0.95)}], lr=1e-3, weight_decay=0.1)
    x, m, v, steps = [t.detach().double() for t in p], [0 * t.detach().double() for t in p], [0 * t.detach().double() for t in p], [0, 0, 0]
    for t in range(10):
        opt.zero_grad()
        for k in range(3):
            if k == 1 and t % 3 == 2:
                continue
            p[k].grad = torch.randn_like(p[k])
            steps[k] += 1
            (x[k], m[k], v[k]), _ = reference(x[k], p[k].grad.double(), m[k], v[k], steps[k], 1e-2 if k < 2 else 1e-3,
                                              (0.9, 0.999) if k < 2 else (0.8, 0.95), 1e-8, 0.1)
        opt.step()
    for k in range(3):
        assert opt.state[p[k]]["step"] == steps[k]
        assert bool(((p[k].double() - x[k]).abs() <= 10 * 20 * U * (x[k].abs() + 1)).all())


@pytest.mark.parametrize("state_bits", [8, 32])
def test_optimiser_state_survives(state_bits):
    from landmark_b200.optim import AdamW

    def model():
        torch.manual_seed(1)
        return [torch.nn.Parameter(torch.randn(n, device="cuda").to(d)) for n, d in ((500, torch.float32), (300, torch.bfloat16), (77, torch.bfloat16))]

    def run(p, opt, first, last):
        for t in range(first, last):
            for k, q in enumerate(p):
                gen = torch.Generator(device="cuda").manual_seed(100 * t + k)
                q.grad = torch.randn(q.shape, generator=gen, device="cuda").to(q.dtype)
            opt.step()

    a = model()
    opt = AdamW(a, lr=1e-2, state_bits=state_bits, seed=5)
    run(a, opt, 0, 3)
    saved = copy.deepcopy(opt.state_dict())
    middle = [q.detach().clone() for q in a]
    run(a, opt, 3, 6)
    b = [torch.nn.Parameter(q) for q in middle]
    again = AdamW(b, lr=1e-2, state_bits=state_bits, seed=5)
    again.load_state_dict(saved)
    s = again.state[b[1]]
    assert s["master"].dtype == torch.float32 and s["exp_avg"].dtype == (torch.float8_e4m3fn if state_bits == 8 else torch.float32)
    run(b, again, 3, 6)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert all(torch.equal(opt.state[x]["exp_avg"].float(), again.state[y]["exp_avg"].float()) for x, y in zip(a, b))
    # parameters that are given other memory, as by a module's .to(), are followed
    a[0].data = a[0].data.clone()
    run(a, opt, 6, 7)
    run(b, again, 6, 7)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_state_of_torch_adamw_is_taken():
    """Five steps of torch's AdamW, then five of this one with its state, against ten in 64 bits (tolerance as above, torch's step rounds no
    more often)."""
    from landmark_b200.optim import AdamW

    torch.manual_seed(3)
    p = [torch.nn.Parameter(torch.randn(n, device="cuda")) for n in (700, 33)]
    x, m, v = ([f(t.detach().double()) for t in p] for f in (torch.clone, torch.zeros_like, torch.zeros_like))
    opt = torch.optim.AdamW(p, lr=1e-2, weight_decay=0.1)
    for t in range(10):
        if t == 5:
            mine = AdamW(p, lr=1e-2, weight_decay=0.1)
            mine.load_state_dict(opt.state_dict())
            opt = mine
        for k in range(2):
            p[k].grad = torch.randn_like(p[k])
            (x[k], m[k], v[k]), _ = reference(x[k], p[k].grad.double(), m[k], v[k], t + 1, 1e-2, (0.9, 0.999), 1e-8, 0.1)
        opt.step()
    for k in range(2):
        assert bool(((p[k].double() - x[k]).abs() <= 10 * 20 * U * (x[k].abs() + 1)).all())


@pytest.mark.parametrize("state_bits", [8, 32])
def test_copied_and_saved_optimisers_go_on(state_bits):
    import io
    import pickle

    from landmark_b200.optim import AdamW

    p = torch.nn.Parameter(torch.randn(600, device="cuda"))
    opt = AdamW([p], lr=1e-2, state_bits=state_bits, seed=4)
    g = torch.randn(600, device="cuda")
    p.grad = g.clone()
    opt.step()

    def saved_and_loaded():
        file = io.BytesIO()
        torch.save(opt.state_dict(), file)
        file.seek(0)
        new = AdamW([torch.nn.Parameter(p.detach().clone())], lr=1e-2, state_bits=state_bits, seed=4)
        new.load_state_dict(torch.load(file))
        return new

    ways = [lambda: copy.deepcopy(opt), saved_and_loaded]
    if state_bits == 32:  # (torch cannot pickle float8 tensors outside torch.save)
        ways.append(lambda: pickle.loads(pickle.dumps(opt)))
    for way in ways:
        again = way()
        assert (again.state_bits, again.seed, again.master_weights) == (state_bits, 4, True)
        q = again.param_groups[0]["params"][0]
        kept = p.detach().clone(), copy.deepcopy(opt.state_dict())
        q.grad = g.clone()
        again.step()
        opt.step()
        assert torch.equal(p, q) and q.data_ptr() != p.data_ptr()
        p.data.copy_(kept[0])
        opt.load_state_dict(kept[1])


def test_closures_schedulers_and_loss_scaling():
    """What torch builds on an optimiser: a closure's loss comes back, a scheduler's rate is the one that is used, a scaled loss whose gradients
    are not finite leaves everything as it was."""
    from landmark_b200.optim import AdamW

    p = torch.nn.Parameter(torch.ones(300, device="cuda"))
    opt = AdamW([p], lr=0.5, weight_decay=0.0)
    rate = torch.optim.lr_scheduler.StepLR(opt, step_size=1, gamma=0.5)

    def closure():
        opt.zero_grad()
        loss = p.sum()
        loss.backward()
        return loss

    assert float(opt.step(closure).detach()) == 300.0
    assert float((p.detach() - 0.5).abs().max()) <= 20 * U  # equal gradients: a step is the rate
    rate.step()
    opt.step(closure)
    assert float((p.detach() - 0.25).abs().max()) <= 20 * U
    scaler = torch.amp.GradScaler("cuda", init_scale=2.0 ** 16)
    kept = p.detach().clone(), opt.state[p]["step"]
    opt.zero_grad()
    scaler.scale((p * float("inf")).sum()).backward()
    scaler.step(opt)
    scaler.update()
    assert torch.equal(p, kept[0]) and opt.state[p]["step"] == kept[1]
    opt.zero_grad()
    scaler.scale(p.sum()).backward()
    scaler.step(opt)
    assert opt.state[p]["step"] == kept[1] + 1 and not torch.equal(p, kept[0])


@pytest.mark.parametrize("dtype,grad,master", [MIXES[0], MIXES[2], MIXES[6]])
@pytest.mark.parametrize("eight", [False, True])
def test_clocked_steps(dtype, grad, master, eight):
    """Steps by a clock are the steps by number: the same states bit for bit, parameters within the bound of one step each (the betas'
    powers are running products there)."""
    from landmark_b200.optim import AdamWClock, AdamWTensors

    def build():
        p, g, m, v, x = tensors(SIZES, dtype, grad)
        scales = ()
        if eight:
            m, v, *scales = random_states(SIZES)
        x = x if master else None
        return AdamWTensors(p, m, v, *(scales or (None, None)), x), g, (p, m, v)

    plain, g, a = build()
    clocked, g2, b = build()
    clock = AdamWClock("cuda", lr=1e-2, betas=(0.9, 0.99), weight_decay=0.1, step=5, seed=77)
    grads = [None if k == 3 else t for k, t in enumerate(g)]
    for step in range(6, 12):
        plain.step(grads, step=step, lr=1e-2 if step < 9 else 3e-3, betas=(0.9, 0.99), weight_decay=0.1, seed=77)
        if step == 9:
            clock.set(lr=3e-3)
        clock.advance()
        clocked.step_clocked([None if k == 3 else t for k, t in enumerate(g2)], clock)
        for x, y in zip(a[1] + a[2], b[1] + b[2]):
            assert torch.equal(bits(x), bits(y))
        off = torch.finfo(dtype).eps * (step - 5)  # a rounding that falls the other way, once a step
        assert all(bool(((x.float() - y.float()).abs() <= off * (x.float().abs() + 0.1)).all()) for x, y in zip(a[0], b[0]))


@pytest.mark.parametrize("eight", [False, True])
def test_captured_steps_go_on(eight):
    from landmark_b200.optim import AdamWClock, AdamWTensors

    def build():
        p, g, m, v, _ = tensors(SIZES, torch.float32, torch.float32)
        scales = ()
        if eight:
            m, v, *scales = random_states(SIZES)
        return AdamWTensors(p, m, v, *scales), g, (p, m, v)

    eager, g, a = build()
    graphed, g2, b = build()
    clocks = [AdamWClock("cuda", lr=1e-2, seed=3) for _ in range(2)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        clocks[1].advance()
        graphed.step_clocked(g2, clocks[1])
    for k in range(8):
        for x, y in zip(g, g2):
            x.normal_(0, 1e-3)
            y.copy_(x)
        if k == 4:
            clocks[0].set(lr=1e-3, betas=(0.8, 0.95))
            clocks[1].set(lr=1e-3, betas=(0.8, 0.95))
        if k == 6:
            clocks[0].set(step=1000)
            clocks[1].set(step=1000)
        clocks[0].advance()
        eager.step_clocked(g, clocks[0])
        graph.replay()
        for xs, ys in zip(a, b):
            assert all(torch.equal(bits(x), bits(y)) for x, y in zip(xs, ys))
    assert torch.equal(clocks[0].memory, clocks[1].memory)
    for bad in ({"lr": -1.0}, {"betas": (1.0, 0.9)}, {"eps": 0.0}, {"step": -2}, {"rate": 1.0}):
        with pytest.raises((RuntimeError, TypeError, ValueError)):
            clocks[0].set(**bad)
    assert torch.equal(clocks[0].memory, clocks[1].memory)


def test_memory_that_moved_and_captures_are_refused():
    from landmark_b200.optim import AdamWTensors

    p, g, m, v, _ = tensors([100, 200], torch.float32, torch.float32)
    t = AdamWTensors(p, m, v)
    strided = torch.randn(200, device="cuda")[::2]
    t.step([strided, g[1]], step=1, lr=1e-3)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(graph):
            t.step(g, step=2, lr=1e-3)
    kept = p[0].clone()
    p[0].data = p[0].data.clone()
    with pytest.raises(ValueError, match="other memory"):
        t.step(g, step=2, lr=1e-3)
    assert torch.equal(p[0], kept)
    with pytest.raises(ValueError, match="memory of another"):
        AdamWTensors([p[0], p[0]], [m[0], m[0].clone()], [v[0], v[0].clone()])
    for bad in ([g[0]], [g[0], g[1][:5]], [g[0], g[1].cpu()]):
        with pytest.raises(ValueError):
            AdamWTensors(p, m, v).step(bad, step=1, lr=1e-3)
    with pytest.raises(TypeError):
        AdamWTensors(p, m, v).step([g[0], g[1].bfloat16()], step=1, lr=1e-3)
    with pytest.raises(TypeError):
        AdamWTensors(p, m, v).step([g[0].double(), g[1].double()], step=1, lr=1e-3)
    with pytest.raises(RuntimeError, match="step 0"):
        AdamWTensors(p, m, v).step(g, step=0, lr=1e-3)
    with pytest.raises(RuntimeError, match="eps"):
        AdamWTensors(p, m, v).step(g, step=1, lr=1e-3, eps=0.0)


def test_offsets_past_32_bits():
    from landmark_b200.optim import adamw_step

    n = 2 ** 31 + 1000
    p, g = torch.full((n,), 0.5, dtype=torch.bfloat16, device="cuda"), torch.full((n,), 0.25, dtype=torch.bfloat16, device="cuda")
    (m, v), (ms, vs) = fresh_8bit(n)
    adamw_step([p], [g], [m], [v], step=1, lr=0.25, weight_decay=0.0, exp_avg_scales=[ms], exp_avg_sq_scales=[vs])
    # equal values: every code is the largest one, and the step is the rate
    assert bool((bits(m) == 0x7E).all()) and bool((bits(v) == 0x7E).all())
    assert bool((p == 0.25).all())


@pytest.mark.parametrize("state_bits", [8, 32])
def test_refused_steps_leave_no_state(state_bits):
    """A first step of the class under a capture is refused before it makes states (their zeros and copies would be captured and never
    written); the eager step that follows is the formula's first."""
    from landmark_b200.optim import AdamW

    torch.manual_seed(2)
    p = [torch.nn.Parameter(torch.randn(n, device="cuda").to(d)) for n, d in ((300, torch.float32), (515, torch.bfloat16))]
    x = [q.detach().float().clone() for q in p]
    opt = AdamW(p, lr=1e-2, weight_decay=0.1, state_bits=state_bits)
    for q in p:
        q.grad = torch.randn_like(q)
    calls = []
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(graph):
            opt.step(lambda: calls.append(1))
    assert len(opt.state) == 0 and not calls
    torch.full((1 << 20,), float("nan"), device="cuda")  # what freed memory may hold
    opt.step()
    for q, a in zip(p, x):
        zero = torch.zeros_like(a).double()
        (want, _, _), (tol, _, _) = reference(a.double(), q.grad.double(), zero, zero, 1, 1e-2, (0.9, 0.999), 1e-8, 0.1)
        assert opt.state[q]["step"] == 1
        got = q if q.dtype == torch.float32 else opt.state[q]["master"]
        assert bool(((got.double() - want).abs() <= tol).all())
        assert torch.equal(q, got.to(q.dtype))


@pytest.mark.parametrize("state_bits", [8, 32])
def test_backward_over_stepped_parameters_is_refused(state_bits):
    """A second backward pass over a graph that kept a parameter's old values is an error, as with torch's optimisers; a parameter that
    had no gradient was not written."""
    from landmark_b200.optim import AdamW, AdamWClock, AdamWTensors

    p = [torch.nn.Parameter(torch.randn(300, device="cuda")) for _ in range(3)]
    opt = AdamW(p, state_bits=state_bits)
    losses = [q.square().sum() for q in p]
    losses[0].backward(retain_graph=True)
    losses[1].backward(retain_graph=True)
    opt.step()
    for loss in losses[:2]:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    losses[2].backward()
    if state_bits == 32:
        q, g, m, v = ([t.clone() for t in ts] for ts in tensors([100, 50], torch.float32, torch.float32)[:4])  # (views share their base's count)
        for clocked in (False, True):
            kept = [t.requires_grad_(True).square().sum() for t in q]
            with torch.no_grad():
                made = AdamWTensors(q, m, v)
                before = [t._version for t in q + m + v]
                if clocked:
                    clock = AdamWClock("cuda", lr=1e-3)
                    clock.advance()
                    made.step_clocked([g[0], None], clock)
                else:
                    made.step([g[0], None], step=1, lr=1e-3)
                assert [t._version > b for t, b in zip(q + m + v, before)] == [True, False] * 3
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                kept[0].backward()
            kept[1].backward()


def test_tensors_that_overlap_are_refused():
    """By part, not only from the same address on; tensors that touch are none."""
    from landmark_b200.optim import AdamWTensors

    flat = torch.zeros(1000, device="cuda")
    m, v = ([torch.zeros(100, device="cuda") for _ in range(2)] for _ in range(2))
    AdamWTensors([flat[:100], flat[100:200]], m, v)
    with pytest.raises(ValueError, match=r"params\[1\] lies in the memory of another tensor of the step, params\[0\]"):
        AdamWTensors([flat[:100], flat[99:199]], m, v)
    with pytest.raises(ValueError, match="memory of another"):
        AdamWTensors([flat[300:400], flat[:100]], m, [v[0], flat[350:450]])
    AdamWTensors([flat[300:400], flat[:100], flat[320:320]], m + [m[0][:0]], v + [v[0][:0]])  # one without values lies nowhere
    codes = torch.zeros(600, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    scales = [torch.zeros(2, device="cuda") for _ in range(2)]
    with pytest.raises(ValueError, match="memory of another"):
        AdamWTensors([flat[:300]], [codes[:300]], [codes[299:599]], scales[:1], scales[1:])
    with pytest.raises(ValueError, match="memory of another"):
        AdamWTensors([flat[:300]], [codes[:300]], [codes[300:]], scales[:1], [flat[299:301]])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("eight", [False, True])
def test_tensors_without_values_beside_masters(dtype, eight):
    """One without values, in first or middle place, changes nothing for 16-bit parameters with 32-bit copies; the class too."""
    from landmark_b200.optim import AdamW, AdamWClock, AdamWTensors

    for sizes in ([0, 300], [300, 0, 257], [0, 0, 5, 0]):
        def build(n):
            p, g, m, v, x = tensors(n, dtype, dtype)
            scales = (None, None)
            if eight:
                m, v, *scales = random_states(n)
            return AdamWTensors(p, m, v, *scales, x), g, (p, m, v, x)

        keep = [k for k, n in enumerate(sizes) if n]
        for clocked in (False, True):
            made, g, a = build(sizes)
            if clocked:
                clock = AdamWClock("cuda", lr=1e-2, step=3, seed=1)
                clock.advance()
                made.step_clocked(g, clock)
            else:
                made.step(g, step=4, lr=1e-2, seed=1)
            alone, g, b = build([sizes[k] for k in keep])
            alone.step(g, step=4, lr=1e-2, seed=1)
            for name, (xs, ys) in zip("pmvx", zip(a, b)):
                for k, y in zip(keep, ys):
                    if not eight or name in "px":  # (codes are rounded by a tensor's number)
                        off = 0.0 if not clocked else torch.finfo(xs[k].dtype).eps * (xs[k].double().abs() + 0.1)
                        assert bool(((xs[k].double() - y.double()).abs() <= off).all())
    q = [torch.nn.Parameter(torch.randn(n, device="cuda").to(dtype)) for n in (0, 300, 0, 7)]
    old = [t.detach().clone() for t in q]
    opt = AdamW(q, lr=0.5, weight_decay=0.0, state_bits=8 if eight else 32)
    for t in q:
        t.grad = torch.ones_like(t)
    opt.step()  # equal gradients: a first step is the rate
    for t, a in zip(q, old):
        want = a.double() - 0.5
        assert bool(((t.double() - want).abs() <= 20 * U * (a.double().abs() + 1) + torch.finfo(dtype).eps / 2 * want.abs() * 1.001 + 2.0 ** -25).all())


@pytest.mark.parametrize("dtype,grad,master", [MIXES[0], MIXES[2]])
@pytest.mark.parametrize("eight", [False, True])
def test_a_clock_before_its_first_step_changes_nothing(dtype, grad, master, eight):
    """Not the parameters by decay, not the states, whatever the gradients hold; also after the count has been set back to 0."""
    from landmark_b200.optim import AdamWClock, AdamWTensors

    p, g, m, v, x = tensors(SIZES, dtype, grad)
    scales = [[], []]
    if eight:
        m, v, *scales = random_states(SIZES)
    made = AdamWTensors(p, m, v, *(scales if eight else (None, None)), x if master else None)
    g[3][0] = float("nan")
    everything = p + m + v + scales[0] + scales[1] + x
    kept = [bits(t.contiguous()).clone() for t in everything]
    clock = AdamWClock("cuda", lr=1e-2, weight_decay=0.1)
    made.step_clocked(g, clock)
    clock.set(lr=0.5)
    made.step_clocked(g, clock)
    clock.advance()
    clock.set(step=0)
    made.step_clocked(g, clock)
    assert all(torch.equal(bits(t.contiguous()), k) for t, k in zip(everything, kept))
    clock.advance()
    made.step_clocked(g, clock)
    assert not torch.equal(bits(p[-1].contiguous()), kept[len(SIZES) - 1])


@pytest.mark.parametrize("state_bits", [8, 32])
def test_memory_of_parameters_is_theirs(state_bits):
    """What a parameter leaves behind when it moves is free at once; when it comes back, or lies otherwise, the step follows or refuses."""
    from landmark_b200.optim import AdamW

    n = 4096
    p = torch.nn.Parameter(torch.randn(n, n, device="cuda"))
    other = torch.nn.Parameter(torch.randn(5, device="cuda"))
    opt = AdamW([p, other], lr=1e-2, weight_decay=0.0, state_bits=state_bits)
    p.grad, other.grad = torch.ones_like(p), torch.ones_like(other)
    opt.step()
    p.grad = None
    before = torch.cuda.memory_allocated()
    p.data = p.data.cpu()
    assert before - torch.cuda.memory_allocated() >= 4 * n * n
    opt.step()  # the other goes on
    taken = torch.full((n, n), 7.0, device="cuda")  # perhaps where the parameter was
    p.data = p.data.cuda()
    p.grad = torch.ones_like(p)
    old = p.detach().clone()
    opt.step()
    assert float((old - p.detach() - 1e-2).abs().max()) <= (1e-6 if state_bits == 32 else 2e-3) and bool((taken == 7.0).all())
    assert opt.state[p]["step"] == 2 and opt.state[other]["step"] == 3
    old = p.detach().clone()
    p.data = p.data.t()  # at the same address
    p.grad = torch.ones(n, n, device="cuda").t()
    with pytest.raises(ValueError, match="contiguous"):
        opt.step()
    assert torch.equal(p.detach(), old.t())


def test_sets_of_parameters_that_moved_are_dropped():
    from landmark_b200.optim import AdamW

    p = [torch.nn.Parameter(torch.randn(100, device="cuda")) for _ in range(2)]
    opt = AdamW([{"params": p[:1]}, {"params": p[1:]}])
    for q in p:
        q.grad = torch.ones_like(q)
    opt.step()
    assert len(opt._sets) == 2
    p[0].grad = None
    opt.step()
    assert len(opt._sets) == 2  # without a gradient for once
    p[0].data = p[0].data.cpu()
    opt.step()
    assert len(opt._sets) == 1


def test_8bit_rounding_of_every_size():
    """The mean of the codes over 1024 seeds, as above, for values from the largest of their block down to far below the smallest code: m is
    kept down to nothing; v is kept where its root is one code (2^-9) or more, and below, where 0 is no choice, it is that code in every case
    (2^-18 of the scale's square, less than v's own rounding beside the largest)."""
    from landmark_b200.optim import adamw_step

    n, seeds = 1024, 1024
    y = 448.0 * 2.0 ** (-24.0 * torch.arange(n, device="cuda") / n)  # spread over four blocks, each beginning with the largest
    g = y.view(256, 4).t().reshape(-1).clone()
    g[::BLOCK] = 448.0
    p = torch.zeros(n, device="cuda")
    m_sum, v_sum = torch.zeros(n, dtype=torch.float64, device="cuda"), torch.zeros(n, dtype=torch.float64, device="cuda")
    for seed in range(seeds):
        (m, v), (ms, vs) = fresh_8bit(n)
        adamw_step([p], [g], [m], [v], step=1, lr=0.0, exp_avg_scales=[ms], exp_avg_sq_scales=[vs], seed=seed)
        m_sum += m.double()
        v_sum += v.double() ** 2
    allowed = 6 * 0.5 / math.sqrt(seeds) + 2.0 ** -17
    y = g.double()  # in units of the scale: the block's largest is 448
    width = torch.exp2(torch.floor(torch.log2(y.clamp(2.0 ** -6, 447.9)))) / 8
    assert bool(((m_sum / seeds - y).abs() <= allowed * width + 1e-6 * y).all())
    small = y < 2.0 ** -9
    assert 100 < int(small.sum()) < 400
    assert bool((v_sum[small] == seeds * 2.0 ** -18).all())
    assert bool(((v_sum / seeds - y * y).abs() <= allowed * (2 * y + width) * width + 1e-6 * y * y)[~small].all())


def test_gradients_with_their_sign_to_come():
    """The imaginary part of a conjugate is read with its sign; as a parameter it is refused."""
    from landmark_b200.optim import AdamWTensors

    for n in (1, 200):
        z = torch.randn(n, dtype=torch.complex64, device="cuda").conj()
        p, m, v = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
        assert z.imag.is_neg()
        AdamWTensors([p], [m], [v]).step([z.imag], step=1, lr=0.25, weight_decay=0.0)
        assert torch.equal(torch.sign(p), -torch.sign(z.imag)) and torch.equal(torch.sign(m), torch.sign(z.imag))
        with pytest.raises(ValueError, match="contiguous"):
            AdamWTensors([z.imag], [m], [v])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_weights_loaded_between_steps_are_kept(dtype):
    """What is written to a 16-bit parameter between steps is where its next step starts, whichever way it was written; values that nobody
    wrote go on from their fp32 copies, as they do in a twin that is left alone."""
    from landmark_b200.optim import AdamW

    def build():
        torch.manual_seed(6)
        p = [torch.nn.Parameter(torch.randn(n, device="cuda").to(dtype)) for n in (300, 40)]
        return p, AdamW(p, lr=1e-3, weight_decay=0.0)

    def step(p, opt, t):
        for k, q in enumerate(p):
            q.grad = None if k == 1 and t == 2 else torch.randn(q.shape, generator=torch.Generator(device="cuda").manual_seed(10 * t + k), device="cuda").to(dtype)
        opt.step()

    new = torch.full((300,), 3.0, dtype=dtype, device="cuda")
    flat = torch.nn.Parameter(new.clone())

    def loaded(q):
        with torch.no_grad():
            q.copy_(new)

    def part(q):
        with torch.no_grad():
            q[:100] = new[:100]

    def replaced(q):
        q.data = flat.detach()

    for t0 in (1, 2, 3):  # before the step where the set changes, and after
        for write, written in ((loaded, 300), (part, 100), (replaced, 300)):
            (p, opt), (q, twin) = build(), build()
            for t in range(5):
                if t == t0:
                    write(p[0])
                    start = p[0].detach().clone()
                step(p, opt, t)
                step(q, twin, t)
                if t == t0:
                    m, v = (opt.state[p[0]][k].double() for k in ("exp_avg", "exp_avg_sq"))
                    update = 1e-3 / (1 - 0.9 ** (t + 1)) * m / (torch.sqrt(v) / math.sqrt(1 - 0.999 ** (t + 1)) + 1e-8)
                    want = (start.double() - update)[:written]
                    assert bool(((opt.state[p[0]]["master"].double()[:written] - want).abs() <= 20 * U * (want.abs() + 1)).all())
                assert torch.equal(p[0], opt.state[p[0]]["master"].to(dtype))
                if t < t0 or write is part:
                    assert torch.equal(opt.state[p[0]]["master"][100:], twin.state[q[0]]["master"][100:])
                assert torch.equal(p[1], q[1]) and torch.equal(opt.state[p[1]]["master"], twin.state[q[1]]["master"])
            flat.data = new.clone()
