"""A Qwen2 decoder whose attention runs on this package's paged-KV contexts.

This is the caller side of the hot path: the reference's ``Qwen2ForCausalLM``
(``engine/model.py:254-323``) with the same parameters, the same order of
parameters and the same tensor operations for everything around attention (embedding
lookup, RMSNorm with float32 statistics, the fused ``qkv_proj`` with bias, ``o_proj``,
the SwiGLU MLP with the fused ``gate_up_proj``, residual adds, the final norm and the
tied or separate LM head). The projections stay on cuBLAS through PyTorch; the residual
adds, the RMSNorms and the MLP's ``silu(gate) * up`` are this package's kernels, one launch
each (``ops.add_rms_norm``, ``ops.silu_mul``) where the reference runs eager chains of
eight or more. Attention goes through the context the runner passes in:
with this package's contexts the layer hands the raw ``qkv_proj`` output to
``ctx.attend_qkv``, which applies RoPE fused with the KV append (bit-identical to the
reference's ``apply_rope``) and runs the paged attention kernels. A context without
``attend_qkv`` (the reference's own) gets the reference's split, head views, RoPE and
``ctx.attend`` call (``engine/model.py:241-251``).

:func:`init_random` reproduces the weights the task's configurations are quoted on:
``torch.manual_seed(seed)`` and then ``normal_(0, std)`` over the parameters in the
reference model's ``named_parameters()`` order, drawn on the CPU in float32 and cast.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch
import torch.nn.functional as F

from . import ops


@dataclass(frozen=True)
class Qwen2Config:
    """The architecture numbers of ``engine/model.py:37-86`` (same field names)."""

    vocab_size: int
    hidden_size: int
    intermediate_size: int
    num_layers: int
    num_heads: int
    num_kv_heads: int
    head_dim: int
    rms_norm_eps: float = 1e-6
    rope_theta: float = 1e6
    max_position_embeddings: int = 32768
    tie_word_embeddings: bool = True
    attention_bias: bool = True
    # Rotary layouts the reference does not have: frequencies stretched for contexts past the
    # trained length, pairs side by side, part of each head (None: all of it).
    rope_scaling: ops.RopeScaling | None = None
    rope_interleaved: bool = False
    rotary_dim: int | None = None
    # Decoder layers the reference does not have. qk_norm: each q and k head is RMS-normalised before its
    # rotation. rope_sections: pairs of a head that are turned by each of up to three position axes
    # (time, height, width; see ops.media_positions), one section after another or in turns. num_experts:
    # the MLP is a mixture of that many experts of expert_intermediate_size, experts_per_token of them
    # for each token, weighted by the softmax over the chosen ones (or over all: renormalize_experts=False).
    qk_norm: bool = False
    rope_sections: tuple[int, ...] | None = None
    rope_sections_alternate: bool = False
    num_experts: int = 0
    experts_per_token: int = 2
    expert_intermediate_size: int | None = None
    renormalize_experts: bool = True

    @property
    def q_size(self) -> int:
        return self.num_heads * self.head_dim

    @property
    def kv_size(self) -> int:
        return self.num_kv_heads * self.head_dim

    # Shapes of the two model families the task's configurations use.
    @classmethod
    def qwen2_0_5b(cls, **kw) -> "Qwen2Config":
        """Qwen2.5-0.5B: 24 layers, hidden 896, 14 / 2 heads of 64, MLP 4864, vocab 151936, tied head."""
        base = dict(vocab_size=151936, hidden_size=896, intermediate_size=4864, num_layers=24, num_heads=14,
                    num_kv_heads=2, head_dim=64, tie_word_embeddings=True)
        base.update(kw)
        return cls(**base)

    @classmethod
    def qwen2_7b(cls, **kw) -> "Qwen2Config":
        """Qwen2.5-7B: 28 layers, hidden 3584, 28 / 4 heads of 128, MLP 18944, vocab 152064, separate head."""
        base = dict(vocab_size=152064, hidden_size=3584, intermediate_size=18944, num_layers=28, num_heads=28,
                    num_kv_heads=4, head_dim=128, tie_word_embeddings=False, max_position_embeddings=33024)
        base.update(kw)
        return cls(**base)


def parameter_shapes(cfg: Qwen2Config) -> list[tuple[str, tuple[int, ...]]]:
    """(name, shape) of every parameter in the reference's ``named_parameters()`` order."""
    h, q, kv, inter = cfg.hidden_size, cfg.q_size, cfg.kv_size, cfg.intermediate_size
    out = [("embed_tokens.weight", (cfg.vocab_size, h))]
    for i in range(cfg.num_layers):
        p = f"layers.{i}."
        out.append((p + "input_norm.weight", (h,)))
        out.append((p + "attn.qkv_proj.weight", (q + 2 * kv, h)))
        if cfg.attention_bias:
            out.append((p + "attn.qkv_proj.bias", (q + 2 * kv,)))
        if cfg.qk_norm:
            out.append((p + "attn.q_norm.weight", (cfg.head_dim,)))
            out.append((p + "attn.k_norm.weight", (cfg.head_dim,)))
        out.append((p + "attn.o_proj.weight", (h, q)))
        out.append((p + "post_attn_norm.weight", (h,)))
        if cfg.num_experts:
            e, mid = cfg.num_experts, cfg.expert_intermediate_size or inter
            out.append((p + "mlp.router.weight", (e, h)))
            out.append((p + "mlp.experts.gate_up_proj.weight", (e, 2 * mid, h)))
            out.append((p + "mlp.experts.down_proj.weight", (e, h, mid)))
        else:
            out.append((p + "mlp.gate_up_proj.weight", (2 * inter, h)))
            out.append((p + "mlp.down_proj.weight", (h, inter)))
    out.append(("norm.weight", (h,)))
    if not cfg.tie_word_embeddings:
        out.append(("lm_head.weight", (cfg.vocab_size, h)))
    return out


def init_random(cfg: Qwen2Config, seed: int = 0, std: float = 0.02, dtype: torch.dtype = torch.float16,
                device: torch.device | str = "cuda", unit_norms: bool = False,
                generator_device: str = "cpu") -> dict[str, torch.Tensor]:
    """Random weights: ``manual_seed(seed)``, then ``normal_(0, std)`` per parameter in order.

    With ``generator_device="cpu"`` (the default) the draws are the reference's: the
    global CPU generator in float32, parameter by parameter, so a reference model seeded
    the same way holds the same values. ``unit_norms`` then sets every RMSNorm weight to
    1 (its draw is still made, so the other parameters do not change): the norms' own
    initial value, which keeps a random model's tokens dependent on its context.
    ``generator_device="cuda"`` draws on the GPU instead (fast, for benchmarks whose
    weights only need the right shapes and scale).
    """
    params: dict[str, torch.Tensor] = {}
    if generator_device == "cpu":
        torch.manual_seed(seed)
        gen = None
    else:
        gen = torch.Generator(device=device).manual_seed(seed)
    for name, shape in parameter_shapes(cfg):
        if gen is None:
            t = torch.empty(shape, dtype=torch.float32)
            t.normal_(0.0, std)
        else:
            t = torch.empty(shape, dtype=torch.float32, device=device)
            t.normal_(0.0, std, generator=gen)
        if unit_norms and name.endswith("norm.weight"):
            t.fill_(1.0)
        params[name] = t.to(device=device, dtype=dtype)
    return params


def _split_k(rows: int, weight: torch.Tensor) -> int:
    """How many K slices a decode batch's projection by ``weight`` gets (0: one cuBLAS GEMM).

    A long-K, small-N projection of a few rows (down_proj of the 0.5B shape: K = 4864, N =
    896) runs as cuBLAS's single GEMM on few SMs (8.2-8.4 us at 64-256 rows, measured); cut
    into 4-8 slices of one batched GEMM with float32 partials it takes 3.9-5.1 us, and the
    next norm sums the partials. Large weights (the 7B shape) stay whole: they stream HBM.
    """
    n, k = weight.shape
    if rows > 256 or k < 4 * n or weight.numel() * weight.element_size() > (32 << 20):
        return 0
    s = 8 if rows <= 128 else 4
    return s if k % s == 0 else 0


def _linear_split_k(x: torch.Tensor, weight: torch.Tensor, splits: int) -> torch.Tensor:
    """``F.linear(x, weight)`` as float32 partial sums ``[splits, rows, N]`` of one batched cuBLAS GEMM.

    ``ops.add_rms_norm`` takes them as its ``x``: it adds the slices in order and rounds to
    the model dtype, where ``F.linear`` rounds its output.
    """
    rows, k = x.numel() // x.shape[-1], x.shape[-1]
    n = weight.shape[0]
    xs = x.reshape(rows, splits, k // splits).transpose(0, 1)  # [S, rows, K/S]
    ws = weight.view(n, splits, k // splits).permute(1, 2, 0)  # [S, K/S, N]
    return torch.bmm(xs, ws, out_dtype=torch.float32)


def _rotate_half(x: torch.Tensor) -> torch.Tensor:
    x1, x2 = x.chunk(2, dim=-1)
    return torch.cat([-x2, x1], dim=-1)


class Qwen2Model:
    """``Qwen2ForCausalLM`` over a dict of weight tensors; ``forward(ids, positions, ctx)`` -> hidden states.

    The call surface is the reference's: ``model(input_ids [B, T], positions [B, T], ctx)``
    returns the final-norm hidden states ``[B, T, hidden]``, ``compute_logits`` applies the
    LM head, ``lm_head_weight`` is the matrix it uses (the embedding when tied) and ``cfg``
    the architecture.
    """

    def __init__(self, cfg: Qwen2Config, weights: dict[str, torch.Tensor]) -> None:
        self.cfg = cfg
        self.w = weights
        self.embed = weights["embed_tokens.weight"]
        self.dtype = self.embed.dtype
        self.device = self.embed.device
        self.lm_head_weight = self.embed if cfg.tie_word_embeddings else weights["lm_head.weight"]
        self.layers = []
        mlp = "mlp.experts." if cfg.num_experts else "mlp."
        self.routers: list[torch.Tensor] = []  # with experts: each layer's, its last two weights then being the experts'
        self.head_norms: list[tuple[torch.Tensor, torch.Tensor, float] | None] = []
        for i in range(cfg.num_layers):
            p = f"layers.{i}."
            self.layers.append((weights[p + "input_norm.weight"], weights[p + "attn.qkv_proj.weight"],
                                weights.get(p + "attn.qkv_proj.bias"), weights[p + "attn.o_proj.weight"],
                                weights[p + "post_attn_norm.weight"], weights[p + mlp + "gate_up_proj.weight"],
                                weights[p + mlp + "down_proj.weight"]))
            if cfg.num_experts:
                self.routers.append(weights[p + "mlp.router.weight"])
            self.head_norms.append((weights[p + "attn.q_norm.weight"], weights[p + "attn.k_norm.weight"], cfg.rms_norm_eps)
                                   if cfg.qk_norm else None)
        if cfg.num_experts and not 1 <= cfg.experts_per_token <= min(16, cfg.num_experts):
            raise ValueError(f"experts_per_token {cfg.experts_per_token} of {cfg.num_experts} experts (at most 16)")
        if cfg.rope_sections is not None and not 1 <= len(cfg.rope_sections) <= 3:
            raise ValueError("rope_sections are pairs of one to three axes")
        # One workspace for the experts of all layers, of the largest step so far (zeroed once, reused):
        # steps of one model must not overlap on the GPU, as with the cache's workspaces. Smaller ones
        # that captured steps hold the addresses of stay.
        self._expert_workspaces: list[torch.Tensor] = []
        self._expert_rows = -1  # tokens that the last one holds
        self._expert_captured = 0  # how many of the first ones stay: up to the last that a captured step holds
        self.norm = weights["norm.weight"]
        # The reference's RoPE tables (float32, cast to the model dtype per lookup), built once.
        # Other layouts and scaled frequencies go through ops.rotary_append, which makes the
        # angles in float64 and rounds once; a context without it takes scaled tables.
        self.cos = self.sin = self.rotary = None
        rotary_dim = cfg.head_dim if cfg.rotary_dim is None else cfg.rotary_dim
        if rotary_dim > cfg.head_dim:
            raise ValueError(f"rotary_dim {rotary_dim} is past head_dim {cfg.head_dim}")
        whole = not cfg.rope_interleaved and rotary_dim == cfg.head_dim
        own = cfg.qk_norm or cfg.rope_sections is not None  # only ops.norm_rotary_append does these
        if not whole or own or cfg.rope_scaling is not None:
            self.rotary = ops.Rotary.build(rotary_dim, cfg.rope_theta, cfg.rope_interleaved, cfg.rope_scaling, self.device,
                                           cfg.rope_sections, cfg.rope_sections_alternate)
        if whole and not own:
            self.cos, self.sin = ops.rope_tables(cfg.head_dim, cfg.max_position_embeddings, cfg.rope_theta, self.dtype,
                                                 self.device, cfg.rope_scaling)

    def weight_bytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self.w.values())

    def _attention(self, layer: int, x: torch.Tensor, positions: torch.Tensor, ctx, wqkv, bqkv, wo) -> torch.Tensor:
        cfg = self.cfg
        b, t, _ = x.shape
        qkv = F.linear(x, wqkv, bqkv)
        if self.rotary is not None and (self.cos is None or hasattr(ctx, "attend_rotary")):  # this package's contexts
            if not hasattr(ctx, "attend_rotary"):
                raise TypeError("this model's rotation and norms need a context of this package (attend_rotary)")
            norm = self.head_norms[layer]
            out = (ctx.attend_rotary(layer, qkv, self.rotary, cfg.num_heads) if norm is None else
                   ctx.attend_rotary(layer, qkv, self.rotary, cfg.num_heads, norm))
        elif hasattr(ctx, "attend_qkv"):
            out = ctx.attend_qkv(layer, qkv, self.cos, self.sin, cfg.num_heads)  # [B, Hq, T, d]
        else:  # engine/model.py:241-250 for a context that only has attend()
            q, k, v = qkv.split([cfg.q_size, cfg.kv_size, cfg.kv_size], dim=-1)
            q = q.view(b, t, cfg.num_heads, cfg.head_dim).transpose(1, 2)
            k = k.view(b, t, cfg.num_kv_heads, cfg.head_dim).transpose(1, 2)
            v = v.view(b, t, cfg.num_kv_heads, cfg.head_dim).transpose(1, 2)
            cos, sin = self.cos[positions].unsqueeze(1), self.sin[positions].unsqueeze(1)
            q, k = q * cos + _rotate_half(q) * sin, k * cos + _rotate_half(k) * sin
            out = ctx.attend(layer, q, k, v)
        return F.linear(out.transpose(1, 2).reshape(b, t, cfg.q_size), wo)

    def expert_workspace(self, rows: int) -> torch.Tensor:
        """The experts' workspace, of at least ``rows`` tokens: a larger one is made outside graph captures only.

        An outgrown one is let go unless a capture took it from here; a graph captured around one that
        was taken before needs the caller to hold on to it.
        """
        capturing = torch.cuda.is_current_stream_capturing()
        if rows > self._expert_rows:
            if capturing:
                raise RuntimeError(f"run a step of {rows} tokens before capturing one: the experts' workspace has to grow")
            self._expert_rows = -1
            while len(self._expert_workspaces) > self._expert_captured:
                # Its memory is another's only once the steps up to here are done, whichever stream they ran on.
                self._expert_workspaces.pop().record_stream(torch.cuda.current_stream(self.device))
            cfg, most = self.cfg, max(64, 1 << (rows - 1).bit_length())
            self._expert_workspaces.append(ops.expert_mlp_workspace(
                most, cfg.num_experts, cfg.experts_per_token, cfg.hidden_size,
                cfg.expert_intermediate_size or cfg.intermediate_size, self.device))
            self._expert_rows = most
        if capturing:
            self._expert_captured = len(self._expert_workspaces)
        return self._expert_workspaces[-1]

    def reset_workspaces(self) -> None:
        """Ready the workspaces again after a step that reported a timed-out wait."""
        for ws in self._expert_workspaces:
            ws.zero_()

    def _experts(self, layer: int, x: torch.Tensor, ctx) -> torch.Tensor:
        cfg = self.cfg
        cache = getattr(ctx, "cache", None)
        return ops.expert_mlp(x, self.routers[layer], *self.layers[layer][5:], cfg.experts_per_token,
                              self.expert_workspace(x.numel() // x.shape[-1]), renormalize=cfg.renormalize_experts,
                              status=getattr(cache, "status", None))

    def __call__(self, input_ids: torch.Tensor, positions: torch.Tensor, ctx,
                 media: list[tuple[int, torch.Tensor]] | None = None) -> torch.Tensor:
        return self.forward(input_ids, positions, ctx, media)

    def forward(self, input_ids: torch.Tensor, positions: torch.Tensor, ctx,
                media: list[tuple[int, torch.Tensor]] | None = None) -> torch.Tensor:
        """engine/model.py:266-318: ``x = x + attn(norm(x)); x = x + mlp(norm(x))`` per layer, then the norm.

        ``h`` is the residual stream ``x``; each block's output ``y`` is added into it by the
        next norm's launch (``ops.add_rms_norm``, the reference's rounding), and the MLP's
        ``silu(gate) * up`` is one launch (``ops.silu_mul``). For decode batches of the 0.5B
        shape ``down_proj`` leaves float32 split-K partials that the next norm sums and rounds
        (see :func:`_split_k`). ``media``: rows ``[n, hidden]`` that take the place of the
        embeddings from the packed token ``a`` on, as ``(a, rows)`` pairs.
        """
        eps = self.cfg.rms_norm_eps
        h = F.embedding(input_ids, self.embed)  # a fresh tensor: updated in place below
        for a, rows in media or ():
            h.view(-1, h.shape[-1])[a:a + rows.shape[0]] = rows
        y = None
        rows = h.numel() // h.shape[-1]
        splits = _split_k(rows, self.layers[0][6]) if self.layers and not self.routers else 0
        for i, (n1, wqkv, bqkv, wo, n2, wgu, wd) in enumerate(self.layers):
            x = ops.add_rms_norm(h, n1, eps) if y is None else ops.add_rms_norm(y, n1, eps, residual=h)
            y = self._attention(i, x.view_as(h), positions, ctx, wqkv, bqkv, wo)
            x = ops.add_rms_norm(y, n2, eps, residual=h)
            if self.routers:
                y = self._experts(i, x, ctx)
                continue
            act = ops.silu_mul(F.linear(x, wgu))
            # down_proj: float32 split-K partials for decode batches, summed by the next norm
            y = _linear_split_k(act, wd, splits) if splits else F.linear(act, wd)
        return ops.add_rms_norm(y, self.norm, eps, residual=h).view_as(h)

    def compute_logits(self, hidden: torch.Tensor) -> torch.Tensor:
        return F.linear(hidden, self.lm_head_weight)
