"""Learning appearance codes of a model whose geometry stays.

An ``encode_app`` model has a learned 48-d latent per image (``embedding_app``, app/models/gridnerf_sequential.py:681-682).  An
image that the trainer never saw has no row of its own; ``AppearanceFit`` learns one (or several at once) from rays with known
colours, and on demand the colour network with them.  Density, samples, weights and projected features come from the library's
kernels and are constants of a step; the network runs under autograd between the package's embedding lookup (a row per sample), its
gradient read as a sum (samples into rays), and the optimiser.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from .embedding import embedding_backward
from .gridnerf import B200GridNeRF
from .optim import AdamW


def _encoded(x: torch.Tensor, freqs: int) -> torch.Tensor:
    """app/tools/utils.py:42-48."""
    pts = (x[..., None] * 2.0 ** torch.arange(freqs, dtype=x.dtype, device=x.device)).reshape(*x.shape[:-1], freqs * x.shape[-1])
    return torch.cat([torch.sin(pts), torch.cos(pts)], dim=-1)


class AppearanceFit:
    """Trains rows of ``model.embedding_app`` (``network``: the colour network too) on rays with known colours.

    ``lr``, ``network_lr``: rates of the two; ``betas``, ``weight_decay``, ``state_bits``: of the optimiser (``optim.AdamW``), with the
    reference trainer's betas as default.  With weight decay, rows that no ray names shrink too.  The library renders with what it was
    given last: call ``finish`` before the next render."""

    def __init__(self, model: B200GridNeRF, lr: float = 1e-2, network: bool = False, network_lr: Optional[float] = None,
                 betas: Tuple[float, float] = (0.9, 0.99), weight_decay: float = 0.0, state_bits: int = 32, seed: int = 0):
        if not model.encode_app:
            raise ValueError("the model has no appearance codes (args.encode_app)")
        self.model = model
        self.table = model.embedding_app.weight
        groups = [{"params": [self.table], "lr": lr}]
        if network:
            groups.append({"params": list(model.renderModule.parameters()), "lr": lr if network_lr is None else network_lr})
        self.optimizer = AdamW(groups, betas=betas, weight_decay=weight_decay, state_bits=state_bits, seed=seed)

    def _parameters(self):
        return [p for group in self.optimizer.param_groups for p in group["params"]]

    def render(self, rays: torch.Tensor, codes: torch.Tensor, N_samples: int = -1, white_bg: bool = True) -> torch.Tensor:
        """Colours ``[n, 3]`` of ``rays [n, 6]`` with the appearance code of each, differentiable in what is trained."""
        m = self.model
        if codes.shape != rays.shape[:1] or codes.dtype not in (torch.int64, torch.int32):
            raise ValueError(f"one int64 or int32 code per ray: got {codes.dtype} {tuple(codes.shape)} for rays {tuple(rays.shape)}")
        codes = codes.to(m.device)
        if codes.numel() and not (0 <= int(codes.min()) and int(codes.max()) < self.table.shape[0]):
            raise ValueError(f"codes must be rows of the table of {self.table.shape[0]}")
        n = rays.shape[0]
        if n == 0:
            return torch.empty((0, 3), device=m.device)
        st = m.run_stages(rays, N_samples, white_bg, upto="appearance")
        ray = st["ray_index"][st["app_index"]]
        features, view = st["app_features"].float(), rays.to(m.device).float()[ray, 3:6]
        parts = [features, m.app_latents(codes[ray])]
        if m.view_pe > -1:
            parts.append(view)
        if m.fea_pe > 0:
            parts.append(_encoded(features, m.fea_pe))
        if m.view_pe > 0:
            parts.append(_encoded(view, m.view_pe))
        colour = torch.sigmoid(m.renderModule.mlp(torch.cat(parts, dim=-1)))
        rgb = embedding_backward(st["weight"][st["app_index"]][:, None] * colour, ray, n)
        if white_bg:
            rgb = rgb + (1.0 - st["acc"])[:, None]
        return rgb.clamp(0, 1)

    def step(self, rays: torch.Tensor, colors: torch.Tensor, codes: torch.Tensor, N_samples: int = -1, white_bg: bool = True) -> torch.Tensor:
        """One step on the mean squared colour error of ``rays``; returns it (a scalar on the device, not waited for)."""
        if tuple(colors.shape) != (rays.shape[0], 3) or rays.shape[0] == 0:
            raise ValueError(f"colors {tuple(colors.shape)} for {rays.shape[0]} rays")
        params = self._parameters()
        wanted = [p.requires_grad for p in params]
        with torch.enable_grad():
            try:
                for p in params:
                    p.requires_grad_(True)
                loss = (self.render(rays, codes, N_samples, white_bg) - colors.to(self.model.device)).square().mean()
                for p, g in zip(params, torch.autograd.grad(loss, params)):
                    p.grad = g
            finally:
                for p, w in zip(params, wanted):
                    p.requires_grad_(w)
        self.optimizer.step()
        self.optimizer.zero_grad()
        return loss.detach()

    def finish(self):
        """Hands the trained rows and network to the library."""
        self.model.network_changed()
