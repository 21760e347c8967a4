"""Learning appearance codes: lookup, network, sum into rays, its gradient, the gradient of the rows and the optimiser together.

The gradients are compared with those of the same formula in 64 bits, norm by norm.  Every layer's dot products of K terms are
off by at most K u of the sum of magnitudes, about sqrt(K) of the result where signs are mixed; forward and backward pass go through
K = 198, 128 and 128 twice: 2 (198 + 128 + 128) sqrt(198) 2^-24 = 7.6e-4, and the sums over samples and rays add less.  Bound: 1e-3."""
import copy

import pytest
import torch

from _util import cuda_model, tiny_rays
from landmark_b200 import scenes

pytestmark = pytest.mark.gpu


def scene():
    spec = scenes.tiny_spec(height=24, width=24, n_samples=48, grid=32).lit()
    spec.encode_app = True
    return spec


def formula(model, stages, rays, codes, table, weights, white_bg=True):
    """Colours in 64 bits from the stages that are constants of a step."""
    ray = stages["ray_index"][stages["app_index"]]
    f, view = stages["app_features"].double(), rays.double()[ray, 3:6]

    def pe(x, n):
        pts = torch.stack([x * 2.0 ** k for k in range(n)], dim=-1).flatten(1)
        return torch.cat([pts.sin(), pts.cos()], 1)

    x = torch.cat([f, table[codes[ray]], view, pe(f, model.fea_pe), pe(view, model.view_pe)], 1)
    for k in (0, 2):
        x = torch.relu(x @ weights[k].t() + weights[k + 1])
    x = torch.sigmoid(x @ weights[4].t() + weights[5])
    rgb = torch.zeros((rays.shape[0], 3), dtype=torch.float64, device=rays.device)
    rgb = rgb.index_add(0, ray, stages["weight"].double()[stages["app_index"]][:, None] * x)
    if white_bg:
        rgb = rgb + (1 - stages["acc"].double())[:, None]
    return rgb.clamp(0, 1)


def batch(spec, model, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rays = tiny_rays(spec).cuda()
    codes = torch.tensor([5, 11499, 77], device="cuda")[torch.randint(0, 3, (rays.shape[0],), generator=gen, device="cuda")]
    return rays, torch.rand((rays.shape[0], 3), generator=gen, device="cuda"), codes


@pytest.mark.parametrize("white_bg,mode", [(True, {}), (False, {}), (True, {"mlp_mode": 2, "app_plane_fp16": True, "density_lattice": True})])
def test_gradients_match_the_formula(white_bg, mode):
    from landmark_b200.appearance import AppearanceFit

    spec = scene()
    model = cuda_model(spec, **mode)
    rays, colors, codes = batch(spec, model)
    fit = AppearanceFit(model, network=True)
    params = fit._parameters()
    for p in params:
        p.requires_grad_(True)
    got = fit.render(rays, codes, spec.n_samples, white_bg)
    grads = torch.autograd.grad((got - colors).square().mean(), params)
    stages = model.run_stages(rays, spec.n_samples, white_bg, upto="appearance")
    exact = [p.detach().double().requires_grad_(True) for p in params]
    rgb = formula(model, stages, rays, codes, exact[0], exact[1:], white_bg)
    assert float((rgb - got).detach().abs().max()) <= 1e-5
    loss = (rgb - colors.double()).square().mean()
    for g, ref in zip(grads, torch.autograd.grad(loss, exact)):
        assert float((g.double() - ref).norm()) <= 1e-3 * float(ref.norm())
    named = torch.zeros(model.embedding_app.weight.shape[0], dtype=torch.bool, device="cuda")
    named[[5, 77, 11499]] = True
    assert bool((grads[0][~named] == 0).all()) and bool((grads[0][named] != 0).any(1).all())
    # and with differences of the formula
    with torch.no_grad():
        for row, col in ((5, 0), (11499, 47)):
            h, values = 1e-4, []
            for sign in (1, -1):
                t = exact[0].detach().clone()
                t[row, col] += sign * h
                values.append((formula(model, stages, rays, codes, t, [e.detach() for e in exact[1:]], white_bg) - colors.double()).square().mean())
            diff = float(values[0] - values[1]) / (2 * h)
            assert abs(float(grads[0][row, col]) - diff) <= 1e-3 * float(grads[0][row].norm())


@pytest.mark.parametrize("state_bits", [8, 32])
@pytest.mark.parametrize("network", [False, True])
def test_steps_run_and_reach_the_renderer(network, state_bits):
    from landmark_b200.appearance import AppearanceFit

    spec = scene()
    model = cuda_model(spec)
    twin = copy.deepcopy({k: v.clone() for k, v in model.state_dict().items()})
    rays, colors, codes = batch(spec, model)
    before, _ = model(rays, app_code=77, N_samples=spec.n_samples)
    fit = AppearanceFit(model, network=network, state_bits=state_bits)
    for _ in range(3):
        assert bool(torch.isfinite(fit.step(rays, colors, codes, spec.n_samples)))
    fit.finish()
    assert not any(p.requires_grad for p in model.parameters())
    changed = (model.embedding_app.weight != twin["embedding_app.weight"]).any(1).nonzero().view(-1).tolist()
    assert changed == [5, 77, 11499]
    assert torch.equal(model.renderModule.mlp[0].weight, twin["renderModule.mlp.0.weight"]) == (not network)
    after, _ = model(rays, app_code=77, N_samples=spec.n_samples)
    assert not torch.equal(after["rgb_map"], before["rgb_map"])
    want = fit.render(rays, torch.full_like(codes, 77), spec.n_samples)
    assert float((after["rgb_map"] - want).abs().max()) <= 1e-4  # the renderer's own bar
    # the same steps give the same bits
    again = cuda_model(spec)
    other = AppearanceFit(again, network=network, state_bits=state_bits)
    for _ in range(3):
        other.step(rays, colors, codes, spec.n_samples)
    assert torch.equal(again.embedding_app.weight, model.embedding_app.weight)


def test_rays_that_meet_nothing_and_refusals():
    from landmark_b200.appearance import AppearanceFit

    spec = scene()
    model = cuda_model(spec)
    fit = AppearanceFit(model)
    rays = torch.tensor([[9.0, 9.0, 9.0, 1.0, 0.0, 0.0]] * 5, device="cuda")
    kept = model.embedding_app.weight.clone()
    loss = fit.step(rays, torch.zeros((5, 3), device="cuda"), torch.zeros(5, dtype=torch.long), spec.n_samples)
    assert float(loss) == 1.0 and torch.equal(model.embedding_app.weight, kept)
    for codes in (torch.zeros(4, dtype=torch.long), torch.zeros(5), torch.full((5,), 11500), torch.full((5,), -1)):
        with pytest.raises(ValueError):
            fit.step(rays, torch.zeros((5, 3), device="cuda"), codes, spec.n_samples)
    with pytest.raises(ValueError):
        fit.step(rays, torch.zeros((4, 3), device="cuda"), torch.zeros(5, dtype=torch.long), spec.n_samples)
    assert not model.embedding_app.weight.requires_grad
    with pytest.raises(ValueError, match="encode_app"):
        AppearanceFit(cuda_model(scenes.tiny_spec(height=24, width=24, n_samples=48, grid=32).lit()))
