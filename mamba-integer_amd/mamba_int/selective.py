"""A selective state space model with a float recurrence on ternary projections.

Where the integer runner (``mamba_int.model``) serves models whose recurrence is
dyadic, this one serves those trained with the float recurrence (softplus steps,
exponential decays, SiLU) on BitLinear projections, with a head in 4-bit weights:

    r += x;  q, s = 8 bits of rms_norm(r)              ops.add_rms_norm_quant
    [u | z] = BitLinear(q, s)                          ops.bitlinear (float output)
    u = silu(conv(u))                                  ops.causal_conv
    [dt | B | C] = BitLinear(u);  dt = BitLinear(dt)   ops.bitlinear_f32
    y = scan(u, dt, A, B, C, D) * silu(z)              ops.selective_scan
    x = BitLinear(y)                                   ops.bitlinear_f32
    ...
    logits = W4 rms_norm(r + x)                        ops.add_rms_norm, ops.w4_matvec

A layer may have a gated linear recurrence in the scan's place, one state a channel:

    [r | i] = BitLinear(u)                             ops.bitlinear_f32
    y = gated scan(u, r, i, decay) * silu(z)           ops.gated_scan

Requests of one batch may each have a low-rank adapter beside the input and output
projections (``Adapters``, ops.adapter_add) and draw their tokens with parameters of
their own (``Sampling``, ops.sample_tokens).

The residual r and every row between the kernels is float32.  Prompts of unequal
lengths run as one padded batch; the state of a sequence is its last conv inputs and
its scan state, and a decode step is the same path over one token.

``python -m mamba_int.selective`` runs a synthetic model and prints its rates.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import List, Optional, Sequence, Tuple, Union

import torch

from . import ops
from .params import ModelDims
from .sampling import Sampling

HEAD_GROUP = 64      # weights of the head that share a scale
GATED_RATE = 8.0     # of a gated layer's log decay


@dataclass
class Projection:
    """Ternary weights [n, k] packed with k padded to 64, and their scale."""
    packed: torch.Tensor
    scale: float
    n: int


@dataclass
class SelectiveLayer:
    norm: torch.Tensor        # float32 [d_model]
    w_in: Projection          # d_model -> 2 d_inner: [u | z]
    conv_w: torch.Tensor      # float32 [d_inner, width]
    conv_b: torch.Tensor
    w_x: Projection           # d_inner -> dt_rank + 2 d_state: [dt | B | C]
    w_dt: Projection          # dt_rank -> d_inner
    dt_bias: torch.Tensor     # float32 [d_inner]
    a: torch.Tensor           # float32 [d_inner, d_state], negative
    d: torch.Tensor           # float32 [d_inner]
    w_out: Projection         # d_inner -> d_model


@dataclass
class GatedLayer:
    norm: torch.Tensor        # float32 [d_model]
    w_in: Projection          # d_model -> 2 d_inner: [u | z]
    conv_w: torch.Tensor      # float32 [d_inner, width]
    conv_b: torch.Tensor
    w_gates: Projection       # d_inner -> 2 d_inner: [r | i]
    decay: torch.Tensor       # float32 [d_inner]
    w_out: Projection         # d_inner -> d_model


@dataclass
class Adapters:
    """Low-rank adapters of a model: for every layer the bank beside w_in, (a [bank, rank, d_model],
    b [bank, 2 d_inner, rank]), and the one beside w_out, (a [bank, rank, d_inner], b [bank, d_model,
    rank]), either may be None; scales float32 [bank] (None: 1).  ``ids`` int32 [B]: each
    sequence's adapter, outside [0, bank) for none."""
    w_in: List[Optional[Tuple[torch.Tensor, torch.Tensor]]]
    w_out: List[Optional[Tuple[torch.Tensor, torch.Tensor]]]
    ids: torch.Tensor
    scales: Optional[torch.Tensor] = None


@dataclass
class SelectiveParams:
    dims: ModelDims
    emb: torch.Tensor         # float32 [vocab, d_model]
    layers: List[Union[SelectiveLayer, GatedLayer]]
    norm_f: torch.Tensor
    head: Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]   # ops.pack_w4's [vocab, d_model]


@dataclass
class SelectiveState:
    """Per layer: the last conv inputs float32 [B, width - 1, d_inner], scan state float32 [B, d_inner, d_state]
    ([B, d_inner] of a gated layer)."""
    conv: List[torch.Tensor]
    h: List[torch.Tensor]


def ternary(w: torch.Tensor) -> Projection:
    """Float weights [n, k] as BitLinear quantizes them (absmean scale, round, clamp)."""
    n, k = w.shape
    scale = float(torch.clamp(w.abs().mean(), min=1e-6))
    q = torch.zeros((n, -(-k // 64) * 64), dtype=torch.int8, device=w.device)
    q[:, :k] = torch.clamp(torch.round(w / scale), -1, 1).to(torch.int8)
    return Projection(ops.pack_ternary(q), scale, n)


def quantize_w4(w: torch.Tensor, group: int = HEAD_GROUP):
    """Float weights [n, k] as 4-bit codes with a float16 scale and a zero point a group of
    columns (the group's range in 15 steps), packed for ``ops.w4_matvec``."""
    n, k = w.shape
    ng = -(-k // group)
    full = torch.zeros((n, ng * group), dtype=torch.float32, device=w.device)
    full[:, :k] = w
    g = full.view(n, ng, group)
    lo, hi = g.amin(-1).clamp(max=0.0), g.amax(-1).clamp(min=0.0)
    scale = ((hi - lo) / 15.0).clamp(min=1e-6).half()
    zero = torch.round(-lo / scale.float()).clamp(0, 15)
    codes = (torch.round(g / scale.float().unsqueeze(-1)) + zero.unsqueeze(-1)).clamp(0, 15)
    codes = codes.to(torch.uint8).view(n, ng * group)[:, :k].contiguous()
    return ops.pack_w4(codes, scale, group, zeros=zero.to(torch.uint8))


def random_params(dims: ModelDims, seed: int, device: str = "cuda", width: int = 4, gated: Sequence[int] = ()) -> SelectiveParams:
    """A synthetic model: normal weights (quantized as above), steps between 0.001 and 0.1
    at dt = 0, decays of 1 .. d_state.  ``gated``: the layers with the gated recurrence,
    whose channels' decays lie between 0.9 and 0.999 where the gate is open."""
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    d, D, N, R = dims.d_model, dims.d_inner, dims.d_state, dims.dt_rank

    def randn(*shape):
        return torch.randn(shape, generator=g, device=device)

    layers = []
    for i in range(dims.n_layer):
        if i in gated:
            a = 0.9 + 0.099 * torch.rand(D, generator=g, device=device)
            layers.append(GatedLayer(
                norm=torch.ones(d, device=device), w_in=ternary(randn(2 * D, d) / math.sqrt(d)),
                conv_w=randn(D, width) / math.sqrt(width), conv_b=0.1 * randn(D),
                w_gates=ternary(randn(2 * D, D) / math.sqrt(D)), decay=torch.log(torch.expm1(-torch.log(a) / GATED_RATE)),
                w_out=ternary(randn(d, D) / math.sqrt(D * 2 * dims.n_layer))))
            continue
        step = torch.exp(torch.rand(D, generator=g, device=device) * math.log(100.0) + math.log(1e-3))
        layers.append(SelectiveLayer(
            norm=torch.ones(d, device=device), w_in=ternary(randn(2 * D, d) / math.sqrt(d)),
            conv_w=randn(D, width) / math.sqrt(width), conv_b=0.1 * randn(D),
            w_x=ternary(randn(R + 2 * N, D) / math.sqrt(D)), w_dt=ternary(randn(D, R) / math.sqrt(R)),
            dt_bias=torch.log(torch.expm1(step)),
            a=-torch.arange(1, N + 1, device=device).float().expand(D, N).contiguous(), d=torch.ones(D, device=device),
            w_out=ternary(randn(d, D) / math.sqrt(D * 2 * dims.n_layer))))
    return SelectiveParams(dims, randn(dims.vocab_size, d), layers, torch.ones(d, device=device),
                           quantize_w4(randn(dims.vocab_size, d) / math.sqrt(d)))


class SelectiveRunner:
    """Prefill, recurrent decode and greedy generation."""

    def __init__(self, params: SelectiveParams):
        dims = params.dims
        dims.validate()
        if dims.ssd or (dims.dt_rank + 2 * dims.d_state) % 4:
            raise ValueError("SelectiveRunner takes dims of the dyadic block's kind, dt_rank + 2 d_state a multiple of 4")
        self.params, self.dims = params, dims
        self.device = params.emb.device

    def new_state(self, batch: int) -> SelectiveState:
        D, N = self.dims.d_inner, self.dims.d_state
        width = self.params.layers[0].conv_w.shape[1]
        return SelectiveState([torch.zeros((batch, width - 1, D), device=self.device) for _ in self.params.layers],
                              [torch.zeros((batch, D) if isinstance(ly, GatedLayer) else (batch, D, N), device=self.device)
                               for ly in self.params.layers])

    @torch.no_grad()
    def forward(self, ids: torch.Tensor, state: SelectiveState, lens: Optional[torch.Tensor] = None,
                adapters: Optional[Adapters] = None) -> torch.Tensor:
        """Logits float32 [B, vocab] of each sequence's last token; ids int64 [B, L], state is
        updated in place.  lens int32 [B]: tokens of each sequence, taken as within [0, L] (the
        rest of its row is padding); one of no tokens has logits of zero.  ``adapters``: each
        sequence's own beside the projections."""
        B, L = ids.shape
        if L < 1:
            raise ValueError("ids must hold at least one token a sequence")
        dims, D, N, R = self.dims, self.dims.d_inner, self.dims.d_state, self.dims.dt_rank
        r = self.params.emb[ids.reshape(-1)]
        x = None
        for i, ly in enumerate(self.params.layers):
            if x is None:
                q, s, _ = ops.add_rms_norm_quant(r, ly.norm)
            else:
                q, s, _ = ops.add_rms_norm_quant(x, ly.norm, residual=r, residual_out=r)
            uz = ops.bitlinear(q, ly.w_in.packed, ops.OUT_FLOAT, 2 * D, x_scale=s, w_scale=ly.w_in.scale).view(B, L, 2 * D)
            if adapters is not None and adapters.w_in[i] is not None:
                a, b = adapters.w_in[i]
                ops.adapter_add(uz, q.view(B, L, -1)[..., :dims.d_model], a, b, adapters.ids, scales=adapters.scales,
                                x_scale=s.view(B, L), lens=lens, out=uz)
            u = ops.causal_conv(uz[..., :D], ly.conv_w, bias=ly.conv_b, state_in=state.conv[i], state_out=state.conv[i],
                                lens=lens)
            if isinstance(ly, GatedLayer):
                ri = ops.bitlinear_f32(u.view(B * L, D), ly.w_gates.packed, ly.w_gates.scale).view(B, L, 2 * D)
                y = ops.gated_scan(u, ri[..., :D], ri[..., D:], ly.decay, z=uz[..., D:], rate=GATED_RATE, h_in=state.h[i],
                                   h_out=state.h[i], lens=lens)
            else:
                xp = ops.bitlinear_f32(u.view(B * L, D), ly.w_x.packed, ly.w_x.scale)
                dt = ops.bitlinear_f32(xp[:, :R].contiguous(), ly.w_dt.packed, ly.w_dt.scale).view(B, L, D)
                xp = xp.view(B, L, R + 2 * N)
                y = ops.selective_scan(u, dt, ly.a, xp[..., R:R + N], xp[..., R + N:], d_skip=ly.d, z=uz[..., D:],
                                       dt_bias=ly.dt_bias, h_in=state.h[i], h_out=state.h[i], lens=lens)
            x = ops.bitlinear_f32(y.view(B * L, D), ly.w_out.packed, ly.w_out.scale)
            if adapters is not None and adapters.w_out[i] is not None:
                a, b = adapters.w_out[i]
                rows = x.view(B, L, -1)
                ops.adapter_add(rows, y, a, b, adapters.ids, scales=adapters.scales, lens=lens, out=rows)
        # a row of its own sequence, whatever lens holds
        last = (lens.clamp(1, L).long() if lens is not None else torch.full((B,), L, device=self.device)) - 1
        rows = last + L * torch.arange(B, device=self.device)
        y, _ = ops.add_rms_norm(x[rows], self.params.norm_f, residual=r[rows])
        if lens is not None:
            y.masked_fill_((lens < 1).unsqueeze(1), 0.0)
        packed, scales, zeros = self.params.head
        return ops.w4_matvec(y, packed, scales, dims.vocab_size, HEAD_GROUP, zeros=zeros)

    @torch.no_grad()
    def generate(self, ids: torch.Tensor, steps: int, lens: Optional[torch.Tensor] = None, sampling: Optional[Sampling] = None,
                 adapters: Optional[Adapters] = None) -> torch.Tensor:
        """Tokens int64 [B, steps] after the prompts: the largest logit's, or drawn as ``sampling``
        says.  A sequence whose logits hold nothing to draw (NaN and -inf alone) ends: it has -1
        from there on."""
        state = self.new_state(ids.shape[0])
        out, logits = [], self.forward(ids, state, lens, adapters)
        for i in range(steps):
            if sampling is None:
                tok = logits.argmax(-1, keepdim=True)
                out.append(tok)
            else:
                tok = sampling.draw(logits).unsqueeze(-1)
                out.append(torch.where(out[-1] < 0, -1, tok) if out else tok)
                tok = out[-1].clamp(min=0)      # (what an ended sequence goes on with is dropped)
            if i + 1 < steps:
                logits = self.forward(tok, state, adapters=adapters)
        return torch.cat(out, 1) if out else ids.new_empty((ids.shape[0], 0))


def main() -> None:
    import time
    dims = ModelDims(d_model=768, n_layer=24, vocab_size=32000, d_state=16, dt_rank=48)
    run = SelectiveRunner(random_params(dims, 1))
    B, L, steps = 8, 2048, 32
    ids = torch.randint(0, dims.vocab_size, (B, L), device=run.device)
    for _ in range(2):
        state = run.new_state(B)
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        logits = run.forward(ids, state)
        torch.cuda.synchronize()
        t1 = time.perf_counter()
        for _ in range(steps):
            logits = run.forward(logits.argmax(-1, keepdim=True), state)
        torch.cuda.synchronize()
        t2 = time.perf_counter()
    print(f"d768 x 24, batch {B}: prefill of {L} tokens {1e3 * (t1 - t0):.2f} ms ({B * L / (t1 - t0):.0f} tok/s), "
          f"decode {1e3 * (t2 - t1) / steps:.3f} ms a step ({B * steps / (t2 - t1):.0f} tok/s)")


if __name__ == "__main__":
    main()
