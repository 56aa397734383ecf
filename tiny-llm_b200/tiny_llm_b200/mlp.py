"""Gated feed-forward layers with unquantised weights: ``down(act(gate x) * (up x))``.

``GatedMLP`` is the dense form (gate and up stacked into one product, the activation fused with the gating product in
one launch); ``TopKRouter`` + ``MixtureOfExperts`` the sparse one: router logits in fp32, the ``top`` largest chosen,
weights either a softmax over the chosen logits or each chosen logit's sigmoid as it is, the chosen experts' outputs
summed with those weights (or, ``weight_on="input"``, each expert run on its weight times the token), optionally plus
a shared expert that every token takes (as it is, or times a sigmoid of a projection of the token).  The choice may be
limited to the best ``groups`` of neighbouring experts.  Experts are gated or, without ``w_gate``, plain ``down(act(up x))``.  The expert products are grouped GEMMs of the blocks library over a device-built
list of (token, choice) pairs sorted by expert: no host synchronisation, and a token's result does not depend on the
rest of the batch."""

from __future__ import annotations

import torch

from .basics import linear, linear_wide

ACTIVATIONS = {"silu": 0, "gelu_tanh": 1, "relu_squared": 2, "clamped_swish": 3}
SCORINGS = {"softmax": 0, "sigmoid": 1, "softmax_all": 2}


class DenseMLP:
    """The ungated feed-forward ``down(act(up x))``; the down projection hands its fp32 accumulator on."""

    def __init__(self, w_up: torch.Tensor, w_down: torch.Tensor, act: str):
        self.w_up, self.w_down, self.act = w_up.contiguous(), w_down.contiguous(), ACTIVATIONS[act]

    def __call__(self, h: torch.Tensor) -> torch.Tensor:
        from extensions_b200.tiny_llm_ext_b200 import blocks

        return linear_wide(blocks.act_rows(linear(h, self.w_up), self.act), self.w_down)


class GatedMLP:
    """``act="clamped_swish"`` (with ``limit`` and ``slope``): ``g = min(gate x, limit)``, ``u = clamp(up x, -limit, limit)``,
    ``down(g sigmoid(slope g) (u + 1))``.  ``b_gate`` / ``b_up`` are added by the first product; ``b_down`` is kept for the
    caller (``down_bias``), who adds it where the residual sum is made."""

    def __init__(self, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, act: str, b_gate=None, b_up=None, b_down=None,
                 limit: float = 0.0, slope: float = 1.0):
        self.w_gate_up = torch.cat([w_gate, w_up], dim=0).contiguous()  # [2 ff, D]: one product for both
        self.w_down = w_down.contiguous()
        self.act = ACTIVATIONS[act]
        if (b_gate is None) != (b_up is None):
            raise ValueError("gated feed-forward: biases on both first projections or on neither")
        self.b_gate_up = None if b_gate is None else torch.cat([b_gate, b_up]).contiguous()
        self.down_bias = None if b_down is None else b_down.contiguous()
        self.limit, self.slope = float(limit), float(slope)
        if act == "clamped_swish" and not self.limit > 0:
            raise ValueError("gated feed-forward: the clamped activation needs a positive limit")

    def inner(self, h: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        """``act(gate h) * (up h)``, the down projection's operand; ``out``: the columns of a wider matrix it goes to."""
        from extensions_b200.tiny_llm_ext_b200 import blocks

        first = linear(h, self.w_gate_up) if self.b_gate_up is None else torch.addmm(self.b_gate_up, h, self.w_gate_up.t())
        return blocks.gated_act(first, self.act, self.limit, self.slope, out)

    def __call__(self, h: torch.Tensor, wide: bool = False) -> torch.Tensor:
        """``wide``: hand the down projection's fp32 accumulator back unrounded (when a norm reads it next)."""
        return (linear_wide if wide else linear)(self.inner(h), self.w_down)


class Fp8GatedMLP:
    """``down(act(gate x) * (up x))`` over matrices of 8-bit numbers (``Fp8Weights``): both products in 8 bits, the inner rows fp32 until
    they are rounded as the input's are.  ``act``, ``limit``, ``slope``: see ``GatedMLP``."""

    def __init__(self, w_gate, w_up, w_down, act: str, limit: float = 0.0, slope: float = 1.0):
        from extensions_b200.tiny_llm_ext_b200 import blocks

        from .fp8 import Fp8Weights, interleaved

        if not all(isinstance(w, Fp8Weights) and len(w.shape) == 2 for w in (w_gate, w_up, w_down)):
            raise ValueError("Fp8GatedMLP: three matrices as Fp8Weights")
        if w_gate.shape != w_up.shape or w_down.shape != w_up.shape[::-1] or len({w.device for w in (w_gate, w_up, w_down)}) != 1:
            raise ValueError(f"Fp8GatedMLP: gate {w_gate.shape}, up {w_up.shape} and down {w_down.shape} do not go together")
        if act not in ("silu", "gelu_tanh", "clamped_swish"):
            raise ValueError(f"Fp8GatedMLP: no gated activation {act!r}")
        self.inner_width, self.width = w_up.shape
        self.gate_up, self.down, self._blocks = interleaved(w_gate, w_up), (w_down.values, w_down.scales), blocks
        self.act, self.limit, self.slope = ACTIVATIONS[act], float(limit), float(slope)
        if act == "clamped_swish" and not self.limit > 0:
            raise ValueError("Fp8GatedMLP: the clamped activation needs a positive limit")

    def __call__(self, h: torch.Tensor) -> torch.Tensor:
        return self._blocks.fp8_gated_mlp_of(h, self.gate_up, self.down, self.width, self.inner_width, self.act, self.limit, self.slope)


class TopKRouter:
    def __init__(self, weight: torch.Tensor, bias: torch.Tensor | None, top: int, scoring: str = "softmax", choice_bias: torch.Tensor | None = None,
                 weight_scale: float = 1.0, groups: tuple | None = None):
        """``scoring="softmax_all"``: scores are a softmax over ALL router outputs, the ``top`` are chosen by score +
        ``choice_bias`` (which the weights do not see), the chosen scores are renormalised and times ``weight_scale``.
        ``groups`` = (count, keep): the outputs form ``count`` equal runs of neighbours, and a token chooses among the ``keep`` runs
        whose best choice score is largest."""
        self.weight, self.bias, self.top = weight.contiguous(), None if bias is None else bias.contiguous(), int(top)
        self.scoring = SCORINGS[scoring]
        self.choice_bias, self.weight_scale = None if choice_bias is None else choice_bias.contiguous(), float(weight_scale)
        if (choice_bias is not None or self.weight_scale != 1.0) and scoring != "softmax_all":
            raise ValueError("router: a choice bias and a weight scale go with scoring='softmax_all'")
        if not 0 < self.top <= weight.shape[0]:
            raise ValueError(f"router: top={top} of {weight.shape[0]} experts")
        self.groups = (0, 0) if groups is None else (int(groups[0]), int(groups[1]))
        count, keep = self.groups
        if groups is not None and (count <= 0 or weight.shape[0] % count or not 0 < keep <= count or keep * (weight.shape[0] // count) < self.top):
            raise ValueError(f"router: {keep} of {count} groups of {weight.shape[0]} outputs cannot give {top} choices")

    def __call__(self, h: torch.Tensor, side_w: torch.Tensor | None = None):
        """-> (expert ids int32 [T, top], weights fp32 [T, top]), and with ``side_w [1, D]`` also ``sigmoid(side_w . h)`` fp32 [T]."""
        from extensions_b200.tiny_llm_ext_b200 import blocks

        return blocks.moe_route(h, self.weight, self.bias, self.top, self.scoring, self.choice_bias, self.weight_scale, self.groups, side_w)


class MixtureOfExperts:
    # With use_few_tokens(), the most tokens of a step that goes to the two launches.  They / the chain of launches, us in a replayed graph, bf16: 64 experts of 1408 x 2048, 6 a token,
    # 1 token 38 / 45, 4 79 / 85, 8 113 / 116, 12 140 / 145, 16 158 / 156, 32 197 / 186; with a shared expert 12 154 / 157, 16 172 / 169; 16 experts of 2048 x 4096, 2 a token,
    # 8 106 / 126, 12 133 / 133, 16 144 / 136.  (2 tokens of the first 55 / 54, with the shared expert 75 / 71; called eagerly 56 / 62 and 83 / 88.)
    FEW_TOKENS = 12

    def __init__(self, router: TopKRouter, w_gate: torch.Tensor | None, w_up: torch.Tensor, w_down: torch.Tensor, act: str,
                 shared: GatedMLP | None = None, weight_on: str = "output", identity: int = 0, limit: float = 0.0, slope: float = 1.0,
                 shared_gate: torch.Tensor | None = None):
        """``w_gate, w_up [E, ff, D]``, ``w_down [E, D, ff]`` (the experts stacked); ``w_gate`` None = experts without a gate.
        ``identity``: the router's last ``identity`` outputs are experts without weights whose output is their input.
        ``limit``, ``slope``: of ``act="clamped_swish"`` (see ``GatedMLP``); ``shared_gate [1, D]``: the shared expert's output is
        multiplied by ``sigmoid(shared_gate . x)``."""
        if weight_on not in ("output", "input"):
            raise ValueError(f"weight_on={weight_on!r}")
        self.identity = int(identity)
        if self.identity < 0 or router.weight.shape[0] != w_up.shape[0] + self.identity:
            raise ValueError(f"router outputs ({router.weight.shape[0]}) != experts ({w_up.shape[0]}) + identity experts ({identity})")
        if self.identity and weight_on == "input":
            raise ValueError("identity experts take the router's weight on their output")
        self.router, self.shared, self.scale_input = router, shared, weight_on == "input"
        self.w_gate, self.w_up, self.w_down = None if w_gate is None else w_gate.contiguous(), w_up.contiguous(), w_down.contiguous()
        self.act, self.limit, self.slope = ACTIVATIONS[act], float(limit), float(slope)
        if act == "clamped_swish" and (not self.limit > 0 or w_gate is None):
            raise ValueError("mixture of experts: the clamped activation needs gated experts and a positive limit")
        if shared_gate is not None and (shared is None or shared_gate.numel() != w_up.shape[2]):
            raise ValueError("mixture of experts: a shared gate of [1, width] goes with a shared expert")
        self.shared_gate = None if shared_gate is None else shared_gate.contiguous()
        self.few = None

    def use_few_tokens(self) -> "MixtureOfExperts":
        """Steps of up to ``FEW_TOKENS`` tokens, or as many as one call of ``FewTokenExperts`` takes if that is less, go to it from now on (bf16 experts whose weight is on
        their output; the same definition, sums in another order and inner rows of fp32 in place of bf16).  Calls with ``into`` do not: their end is fused with the
        sublayer's.  Experts of odd widths are held twice from then on (``FewTokenExperts``)."""
        if self.scale_input:
            raise ValueError("mixture of experts: the few-token layer takes the router's weight on the experts' output")
        act = next(name for name, code in ACTIVATIONS.items() if code == self.act)
        self.few = FewTokenExperts(self.router, self.w_gate, self.w_up, self.w_down, act, self.shared, self.identity, self.limit, self.slope, self.shared_gate)
        return self

    def __call__(self, h: torch.Tensor, into: tuple | None = None, beside=None) -> torch.Tensor:
        """-> fp32 [T, D], or (``into`` = (stream, post norm, next norm)) the fused end of the sublayer, see ``blocks.moe_experts``.
        ``beside``: a model whose second stream runs the shared expert while this one routes (``RaggedDecoderModel._beside``)."""
        from extensions_b200.tiny_llm_ext_b200 import blocks

        if self.few is not None and into is None and h.shape[0] <= min(self.few.run, self.FEW_TOKENS):
            return self.few(h, wide=True)
        shared = side = None
        if beside is not None and self.shared is not None:
            shared = torch.empty_like(h)
            with beside._beside():
                torch.mm(self.shared.inner(h), self.shared.w_down.t(), out=shared)
        elif self.shared is not None:
            shared = self.shared(h)
        if self.shared_gate is None:
            idx, gate = self.router(h)
        else:
            idx, gate, side = self.router(h, self.shared_gate)
        join = beside._join if beside is not None and self.shared is not None else None
        return blocks.moe_experts(h, idx, gate, self.w_gate, self.w_up, self.w_down, self.act, shared, scale_input=self.scale_input, identity=self.identity > 0,
                                  limit=self.limit, slope=self.slope, shared_gate=side, into=into, before_sum=join)


def _whole_rows(w: torch.Tensor, rows: int) -> torch.Tensor:
    """A stack of matrices with ``rows`` rows of whole 16-byte pieces, zero behind what it holds; itself where it is laid out so."""
    per = 16 // w.element_size()
    n, k = w.shape[1:]
    if n == rows and k % per == 0 and w.is_contiguous() and w.data_ptr() % 16 == 0:
        return w
    wide = torch.zeros((w.shape[0], rows, -(-k // per) * per * w.element_size()), dtype=torch.uint8, device=w.device).view(w.dtype)
    wide.view(torch.uint8)[:, :n, : k * w.element_size()] = w.contiguous().view(torch.uint8)
    return wide


class FewTokenExperts:
    """A whole mixture-of-experts layer for the few tokens of a decoding step in two launches: router and first products, second products
    and their sum.  Arguments as ``MixtureOfExperts`` takes them, the experts bf16 ``[E, ff, D]`` / ``[E, D, ff]`` or ``Fp8Weights`` of those shapes; the
    router's weight is on the experts' output.  A step of more tokens than one call takes (``run``, see ``blocks.moe_few_tokens``: at most 32, fewer of wide rows, over
    bf16 experts, with many router outputs or choices; sizes that take none are refused) is several calls, each of which reads its experts anew: prompts are better served
    by ``MixtureOfExperts``.  Matrices whose rows are no whole 16-byte pieces (or, of ``w_down``, whose number of rows is no multiple of 8) are copied into such rows when the layer is made: a
    second copy of the experts, which later writes to the first do not reach.  Inner rows are fp32;
    8-bit experts use all but 2^-12 of a number of theirs where the output is bf16 (``wide``: 2^-24), and of a token what lies above 2^-21 of its largest magnitude."""

    def __init__(self, router: TopKRouter, w_gate, w_up, w_down, act: str, shared: GatedMLP | None = None, identity: int = 0, limit: float = 0.0, slope: float = 1.0,
                 shared_gate: torch.Tensor | None = None):
        from extensions_b200.tiny_llm_ext_b200 import blocks

        from .fp8 import Fp8Weights

        weights = [w for w in (w_gate, w_up, w_down) if w is not None]
        fp8 = isinstance(w_up, Fp8Weights)
        if any(isinstance(w, Fp8Weights) != fp8 for w in weights) or any(len(w.shape) != 3 for w in weights):
            raise ValueError("FewTokenExperts: stacks of matrices, all of 8 bits or none")
        E, ff, D = w_up.shape
        if tuple(w_down.shape) != (E, D, ff) or (w_gate is not None and tuple(w_gate.shape) != (E, ff, D)):
            raise ValueError(f"FewTokenExperts: up {tuple(w_up.shape)} and down {tuple(w_down.shape)} do not go together")
        if not fp8 and any(w.dtype != torch.bfloat16 for w in weights):
            raise ValueError("FewTokenExperts: unquantised experts must be bfloat16")
        if identity < 0 or router.weight.shape != (E + identity, D) or router.weight.dtype != torch.bfloat16:
            raise ValueError(f"FewTokenExperts: the router must be bfloat16 [{E} experts + {identity} identity experts, {D}]")
        if (act == "relu_squared" and w_gate is not None) or (act == "clamped_swish" and (w_gate is None or not limit > 0)):
            raise ValueError(f"FewTokenExperts: activation {act!r} does not go with {'gated' if w_gate is not None else 'ungated'} experts")
        if shared_gate is not None and (shared is None or shared_gate.numel() != D):
            raise ValueError("FewTokenExperts: a shared gate of [1, width] goes with a shared expert")
        if len({w.device for w in (*weights, router.weight)}) != 1:
            raise ValueError("FewTokenExperts: router and experts on two devices")
        self.router, self.shared, self.width = router, shared, D
        self._pad = -D % 8
        rows = D + self._pad
        raw = lambda w, n: None if w is None else _whole_rows(w.values if fp8 else w.contiguous(), n)  # noqa: E731
        wider = lambda t: t if t is None or not self._pad else torch.nn.functional.pad(t.reshape(-1, D), (0, self._pad)).contiguous()  # noqa: E731
        self._few = blocks.MoeFew(wider(router.weight), router.bias, router.top, raw(w_gate, ff), raw(w_up, ff), raw(w_down, rows), ACTIVATIONS[act],
                                  scales=None if not fp8 else tuple(None if w is None else w.scales for w in (w_gate, w_up, w_down)), inner=ff, scoring=router.scoring,
                                  choice_bias=router.choice_bias, weight_scale=router.weight_scale, groups=router.groups,
                                  side_w=None if shared_gate is None else wider(shared_gate.contiguous()), limit=limit, slope=slope)
        self.run = self._few.tokens
        if self.run == 0:
            raise ValueError(f"FewTokenExperts: width {D}, {E + identity} router outputs and {router.top} choices do not fit")

    def __call__(self, h: torch.Tensor, wide: bool = False) -> torch.Tensor:
        """``h [T, D]`` bf16 -> ``[T, D]`` bf16, or with ``wide`` the fp32 sums."""
        shared = None if self.shared is None else self.shared(h)
        if self._pad:
            if h.dim() != 2 or h.shape[1] != self.width:
                raise RuntimeError(f"FewTokenExperts: expected bfloat16 [tokens, {self.width}]")
            h, shared = (None if t is None else torch.nn.functional.pad(t, (0, self._pad)) for t in (h, shared))
        if not h.is_contiguous() or h.data_ptr() % 16:
            h = h.clone(memory_format=torch.contiguous_format)
        T = h.shape[0]
        if T <= self.run:
            y = self._few(h, shared, wide)
        else:
            y = torch.cat([self._few(h[t : t + self.run], None if shared is None else shared[t : t + self.run], wide) for t in range(0, T, self.run)])
        return y[:, : self.width].contiguous() if self._pad else y  # the norm behind reads whole rows
