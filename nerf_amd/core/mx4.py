"""A radiance field that answers in microscaled 4-bit numbers.

`Mx4NeRF(nerf)` is a frozen copy of a trained field: every Linear's weight packed once with `ops.mx4_quantize` (4.25 bits
a weight), every layer one `ops.mx4_linear` whose input was quantised on its way out of the layer before.  Activations
take 4.25 bits a value in memory, sums are fp32, biases and both output activations too.  It goes wherever a field goes
that is not trained: `forward`, `BoundedVolumeRaymarcher.render_volume(train=False)`, `nerf_amd.infer`.  Its layers are
calls of their own, so that the width is not bound to what the fused kernels of `NeRF` hold on chip (256): a wider field, for
which there are no such kernels, is served this way.  Up to 256 the bf16 kernels are faster and closer; there it saves memory only.

It is a coarse form: encoded points, activations and weights are all rounded to 4 bits, and nothing trains or calibrates the field
for it.  Against the fp32 frame a field as it is made has 49 dB (bf16: 88), one after 2,000 steps on a smooth pattern 19 dB (bf16: 57)."""
import copy
from typing import Optional, Tuple

import torch
from torch import Tensor
from torch.nn import Linear, Module, ModuleList, Parameter

from .. import ops
from .activations import shifted_softplus, widened_sigmoid

_ACTS = {"ReLU": "relu", "LeakyReLU": "leaky_relu", "SiLU": "silu"}
CHUNK = 1 << 20          # samples that a render works on at a time: 136 bytes each and layer at width 256


class Mx4Linear(Module):
    """A frozen `torch.nn.Linear` with its weight in 4 bits.  `split`: the input is given as two blocks, columns [split:] of
    the layer's input first and columns [:split] behind them (blocks of 32 have to begin where a part begins)."""

    def __init__(self, linear: Linear, split: int = 0) -> None:
        super().__init__()
        w = linear.weight.detach()
        parts = [w] if split == 0 else [w[:, split:], w[:, :split]]
        packed = ops.Mx4.cat([ops.mx4_quantize(p) for p in parts])
        self.in_features, self.out_features, self.split = w.shape[1], w.shape[0], split
        self.register_buffer("codes", packed.codes)
        self.register_buffer("scales", packed.scales)
        self.bias = None if linear.bias is None else Parameter(linear.bias.detach().float().clone(), requires_grad=False)

    @property
    def weight(self) -> "ops.Mx4":
        return ops.Mx4(self.codes, self.scales, self.in_features)

    def forward(self, x, activation: Optional[str] = None, out_dtype=None):
        return ops.mx4_linear(x, self.weight, self.bias, activation, out_dtype)


class Mx4NeRF(Module):
    """The 4-bit form of a `NeRF` (width a multiple of 32), on the device its weights are on."""

    def __init__(self, nerf) -> None:
        super().__init__()
        name = ops.activation_name(nerf)
        if name not in _ACTS:
            raise NotImplementedError(f"hidden activation {name} has no 4-bit form (ReLU / LeakyReLU / SiLU)")
        if name == "LeakyReLU" and abs(float(ops.child(nerf, "fc_1", "0", "1").negative_slope) - 0.01) > 1e-12:
            raise NotImplementedError("LeakyReLU kernels use the default negative_slope=0.01")
        if nerf.width % 32:
            raise ValueError(f"a 4-bit field's width is a multiple of 32 (got {nerf.width})")
        self.phi_x, self.phi_d = copy.deepcopy(nerf.phi_x), copy.deepcopy(nerf.phi_d)
        self.width, self.depth, self.resid, self.activ = nerf.width, nerf.depth, nerf.resid, _ACTS[name]
        linear = lambda block: ops.child(block, "0")
        skip = nerf.phi_x.o_dim if nerf.resid else 0
        with torch.no_grad():
            self.fc_1 = ModuleList(Mx4Linear(linear(b)) for b in nerf.fc_1)
            self.fc_2 = ModuleList(Mx4Linear(linear(b), skip if i == 0 else 0) for i, b in enumerate(nerf.fc_2))
            self.sigma = Mx4Linear(linear(nerf.sigma))
            self.features = Mx4Linear(nerf.features)
            self.rgb = ModuleList((Mx4Linear(ops.child(nerf.rgb, "0"), nerf.phi_d.o_dim), Mx4Linear(ops.child(nerf.rgb, "2"))))

    def _answer(self, px: "ops.Mx4", pd: Optional["ops.Mx4"]) -> Tuple[Tensor, Optional[Tensor]]:
        """Encoded points (and directions, or None: density only) -> sigma (M,), rgb (M, 3)."""
        h = px
        for layer in self.fc_1:
            h = layer(h, self.activ, "mx4")
        for i, layer in enumerate(self.fc_2):
            h = layer(ops.Mx4.cat((h, px)) if i == 0 and self.resid else h, self.activ, "mx4")
        sigma = shifted_softplus(self.sigma(h, out_dtype=torch.float32)).view(-1)
        if pd is None:
            return sigma, None
        c = self.rgb[0](ops.Mx4.cat((self.features(h, None, "mx4"), pd)), self.activ, "mx4")
        return sigma, widened_sigmoid(self.rgb[1](c, out_dtype=torch.float32))

    @torch.no_grad()
    def forward(self, rx: Tensor, rd: Tensor) -> Tuple[Tensor, Tensor]:
        """rx, rd (..., 3) -> sigma (M,), rgb (..., 3) with M = prod(leading dims), as `NeRF.forward`; no graph."""
        x, d = rx.detach().reshape(-1, 3), rd.detach().reshape(-1, 3)
        assert x.shape == d.shape, "positions and directions must pair up"
        sigma, rgb = self._answer(ops.mx4_quantize(self.phi_x(x)), ops.mx4_quantize(self.phi_d(d)))
        return sigma, rgb.reshape(*rx.shape[:-1], 3)

    @torch.no_grad()
    def rays(self, ro: Tensor, rd: Tensor, t: Tensor, density_only: bool = False) -> Tuple[Tensor, Optional[Tensor]]:
        """The field at ro + t rd: ro, rd (B, 3), t (B, n) -> sigma (B, n), rgb (B, n, 3) or None."""
        B, n = t.shape
        sigma = torch.empty((B, n), device=t.device)
        rgb = None if density_only else torch.empty((B, n, 3), device=t.device)
        step = max(1, CHUNK // n)
        for s in range(0, B, step):
            e = min(s + step, B)
            x = ro[s:e, None] + t[s:e, :, None] * rd[s:e, None]
            pd = None
            if not density_only:                                # one direction a ray: encoded once, its codes repeated
                q = ops.mx4_quantize(self.phi_d(rd[s:e]))
                pd = ops.Mx4(q.codes.repeat_interleave(n, 0), q.scales.repeat_interleave(n, 0), q.k)
            a, c = self._answer(ops.mx4_quantize(self.phi_x(x.view(-1, 3))), pd)
            sigma[s:e] = a.view(-1, n)
            if c is not None:
                rgb[s:e] = c.view(-1, n, 3)
        return sigma, rgb
