"""FitLLM's own LoRA wrapper API (fitllm/lora.py:12-138), B200 edition.

``LoRALinear(base, rank, alpha)`` keeps the reference layout -- ``lora_A``
[in, r] ~ N(0, 0.02), ``lora_B`` [r, out] zeros, ``scale = alpha / rank``,
``forward = base(x) + (x @ A @ B) * scale`` -- and ``LoRAManager`` keeps
``inject_lora`` / ``state_dict`` / ``load_state_dict`` /
``trainable_parameters`` / ``freeze_base_model``.

When the wrapped base is an NF4 ``Linear4bit`` the whole expression runs as
one fused QLoRA call on the sm_100a kernels (the adapter is handed over as the
transposed views A^T [r, in] and B^T [out, r]).  A dense ``nn.Linear`` base
(the reference's unquantised test models) keeps the reference's plain torch
arithmetic, since there is no NF4 weight to stream.

``MultiLoRAManager`` serves many trained adapters on one model: each sequence of a
batch takes its own (``MultiLoRALinear``, ops.multi_lora).
"""
from __future__ import annotations

import logging
import math
from typing import Dict, Iterator, List, Optional, Sequence, Tuple

import torch
import torch.nn as nn
from torch.autograd import forward_ad

from . import ops
from .qlora import Linear4bit, _QLoRAFunction

logger = logging.getLogger(__name__)


class LoRALinear(nn.Module):
    """forward(x) = base(x) + scale * (x @ A @ B), scale = alpha / rank."""

    def __init__(self, base_linear: nn.Module, rank: int, alpha: float) -> None:
        super().__init__()
        self.base = base_linear
        self.rank = rank
        self.alpha = alpha
        self.scale = alpha / rank
        in_features = base_linear.in_features
        out_features = base_linear.out_features
        dev = next(base_linear.parameters()).device if any(True for _ in base_linear.parameters()) else None
        self.lora_A = nn.Parameter(torch.empty(in_features, rank, device=dev))
        self.lora_B = nn.Parameter(torch.zeros(rank, out_features, device=dev))
        nn.init.normal_(self.lora_A, mean=0.0, std=0.02)
        for p in self.base.parameters():
            p.requires_grad_(False)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if isinstance(self.base, Linear4bit):
            if self.rank % 16 == 0 and self.rank <= 64:
                return _QLoRAFunction.apply(x, self.lora_A.t(), self.lora_B.t(), self.base.bias,
                                            self.base.wref(), float(self.scale))
            raise ValueError(f"rank {self.rank}: the NF4 kernels take ranks 16, 32, 48 or 64")
        return self.base(x) + (x @ self.lora_A @ self.lora_B) * self.scale

    def extra_repr(self) -> str:
        return (f"in_features={self.base.in_features}, out_features={self.base.out_features}, "
                f"rank={self.rank}, alpha={self.alpha}")


_LINEAR_TYPES = (nn.Linear, Linear4bit)


class LoRAManager:
    """Injection and persistence of LoRALinear adapters."""

    def __init__(self) -> None:
        self._lora_layers: Dict[str, LoRALinear] = {}

    def inject_lora(self, model: nn.Module, rank: int, alpha: float,
                    targets: Tuple[str, ...] = ("q_proj", "k_proj", "v_proj", "o_proj")) -> nn.Module:
        """Replace every linear (dense or NF4) whose name is, or ends with, a target."""
        self._lora_layers.clear()
        todo: List[Tuple[nn.Module, str, LoRALinear]] = []
        for module_name, module in model.named_modules():
            for child_name, child in module.named_children():
                full = f"{module_name}.{child_name}" if module_name else child_name
                if isinstance(child, _LINEAR_TYPES) and any(
                        child_name == t or full.endswith(t) for t in targets):
                    layer = LoRALinear(child, rank=rank, alpha=alpha)
                    todo.append((module, child_name, layer))
                    self._lora_layers[full] = layer
        for parent, name, layer in todo:
            setattr(parent, name, layer)
        logger.info("Injected LoRA into %d linear layers", len(self._lora_layers))
        return model

    def state_dict(self) -> Dict[str, torch.Tensor]:
        sd: Dict[str, torch.Tensor] = {}
        for name, layer in self._lora_layers.items():
            sd[f"{name}.lora_A"] = layer.lora_A.data.clone()
            sd[f"{name}.lora_B"] = layer.lora_B.data.clone()
        return sd

    def load_state_dict(self, sd: Dict[str, torch.Tensor]) -> None:
        for name, layer in self._lora_layers.items():
            if f"{name}.lora_A" in sd:
                layer.lora_A.data.copy_(sd[f"{name}.lora_A"])
            if f"{name}.lora_B" in sd:
                layer.lora_B.data.copy_(sd[f"{name}.lora_B"])

    def trainable_parameters(self) -> Iterator[nn.Parameter]:
        for layer in self._lora_layers.values():
            yield layer.lora_A
            yield layer.lora_B

    def freeze_base_model(self, model: nn.Module) -> None:
        keep = {id(p) for l in self._lora_layers.values() for p in (l.lora_A, l.lora_B)}
        for p in model.parameters():
            if id(p) not in keep:
                p.requires_grad_(False)

    @property
    def num_lora_layers(self) -> int:
        return len(self._lora_layers)


class AdapterRoute:
    """Which adapter slot each sequence of the running batch uses: ``adapter`` int32 [batch]
    (-1: none) and ``q_start`` int32 [batch + 1] of packed tokens (``tokens`` rows of them in a
    pass), or None where every sequence has as many.  Shared by the layers of a MultiLoRAManager."""

    def __init__(self) -> None:
        self.adapter: Optional[torch.Tensor] = None
        self.q_start: Optional[torch.Tensor] = None
        self.tokens: Optional[int] = None

    def check(self, lead: Sequence[int]) -> None:
        """Raises where a pass over x [*lead, in] is not of the routed sequences (host values only)."""
        if self.adapter is None:
            return
        if self.q_start is None:
            if not lead or lead[0] != self.adapter.shape[0]:
                raise ValueError(f"route: {self.adapter.shape[0]} sequences, the pass has {list(lead)} rows "
                                 "(the first dimension is the batch; packed tokens need q_start)")
        elif self.tokens is not None and math.prod(lead) != self.tokens:
            raise ValueError(f"route: {self.tokens} packed tokens, the pass has {list(lead)} rows")


class MultiLoRALinear(nn.Module):
    """An NF4 Linear4bit with ``slots`` adapters of rank up to ``rank``, one per sequence:
    forward(x) = base(x) + scaling[l] (x.A_l^T).B_l^T, l = the sequence's slot in ``route``.
    The adapters are held in bf16 as the kernels read them, A [slots, rank, in] and B [slots,
    out, rank].  For serving: inputs that require a gradient are refused."""

    def __init__(self, base_layer: Linear4bit, slots: int, rank: int, route: AdapterRoute) -> None:
        super().__init__()
        if rank not in (16, 32, 48, 64):
            raise ValueError(f"rank {rank} unsupported (kernels take 16, 32, 48 or 64; smaller adapters are padded)")
        if slots < 1:
            raise ValueError(f"MultiLoRALinear: slots={slots}")
        if base_layer.in_features % 8 or base_layer.out_features % 8:
            raise ValueError("MultiLoRALinear: in_features and out_features must be multiples of 8")
        self.base_layer, self.slots, self.rank, self.route = base_layer, slots, rank, route
        dev = base_layer.weight.device
        self.register_buffer("lora_A", torch.zeros(slots, rank, base_layer.in_features, dtype=torch.bfloat16, device=dev))
        self.register_buffer("lora_B", torch.zeros(slots, base_layer.out_features, rank, dtype=torch.bfloat16, device=dev))
        self.register_buffer("scaling", torch.zeros(slots, dtype=torch.float32, device=dev))

    @property
    def in_features(self) -> int:
        return self.base_layer.in_features

    @property
    def out_features(self) -> int:
        return self.base_layer.out_features

    @torch.no_grad()
    def load(self, slot: int, lora_a: torch.Tensor, lora_b: torch.Tensor, scaling: float) -> None:
        """Adapter A [r, in], B [out, r] (PEFT layout, r <= rank) into a slot."""
        r = lora_a.shape[0]
        if not 0 <= slot < self.slots:
            raise IndexError(f"slot {slot} of {self.slots}")
        if r > self.rank or lora_a.shape != (r, self.in_features) or lora_b.shape != (self.out_features, r):
            raise ValueError(f"adapter {tuple(lora_a.shape)}, {tuple(lora_b.shape)} does not fit [<= {self.rank}, "
                             f"{self.in_features}], [{self.out_features}, .]")
        self.unload(slot)
        self.lora_A[slot, :r].copy_(lora_a)
        self.lora_B[slot, :, :r].copy_(lora_b)
        self.scaling[slot] = float(scaling)

    @torch.no_grad()
    def unload(self, slot: int) -> None:
        self.lora_A[slot].zero_()
        self.lora_B[slot].zero_()
        self.scaling[slot] = 0.0

    def refuse_gradient(self, *inputs: Optional[torch.Tensor]) -> None:
        """Raises where an input's gradient or tangent would be lost (before the passes' no_grad hides it)."""
        if torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in inputs):
            ops._serving_only("MultiLoRALinear")
        if forward_ad._current_level >= 0:
            ops._refuse_tangents("MultiLoRALinear", *inputs)

    @torch.no_grad()
    def add_adapters(self, x2: torch.Tensor, y2: torch.Tensor) -> torch.Tensor:
        """y2 [tokens, out] (bf16, written over) plus the adapters of x2 [tokens, in], rows of a
        pass that ``route.check`` has seen."""
        route = self.route
        if route.adapter is None:
            return y2
        return ops.multi_lora(x2, self.lora_A, self.lora_B, self.scaling, route.adapter, y2, q_start=route.q_start, out=y2)

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        self.refuse_gradient(x, residual)
        self.route.check(x.shape[:-1])
        with torch.no_grad():
            y = self.base_layer(x, residual=residual)
            y2 = self.add_adapters(ops._bf16_2d(x, self.in_features), ops._bf16_2d(y, self.out_features))
            return y2.view(y.shape).to(y.dtype)

    def extra_repr(self) -> str:
        return f"slots={self.slots}, rank={self.rank}"


class MultiLoRAManager:
    """Adapters of many requests on one model: ``apply`` wraps the target Linear4bit modules,
    ``load`` puts a trained adapter (PEFT names, as QLoRAManager saves them) into a slot, ``route``
    says which sequence of the next passes uses which slot."""

    def __init__(self, slots: int, rank: int = 16,
                 targets: Tuple[str, ...] = ("q_proj", "k_proj", "v_proj", "o_proj")) -> None:
        self.slots, self.rank, self.targets = slots, rank, tuple(targets)
        self.routing = AdapterRoute()
        self.layers: Dict[str, MultiLoRALinear] = {}

    def apply(self, model: nn.Module) -> nn.Module:
        """Wraps every Linear4bit whose name is, or ends with, a target."""
        for mod_name, mod in list(model.named_modules()):
            for child_name, child in list(mod.named_children()):
                full = f"{mod_name}.{child_name}" if mod_name else child_name
                if isinstance(child, Linear4bit) and any(full == t or full.endswith("." + t) for t in self.targets):
                    layer = MultiLoRALinear(child, self.slots, self.rank, self.routing)
                    setattr(mod, child_name, layer)
                    self.layers[full] = layer
        return model

    def load(self, slot: int, state: Dict[str, torch.Tensor], alpha: float) -> int:
        """A state dict with ``...<module>.lora_A(.default).weight`` and ``lora_B`` keys into a
        slot, scaled by alpha / r; returns how many projections it covers, and raises, changing
        nothing, where a pair is incomplete or none matches.  Projections it does not name have none."""
        pairs: Dict[str, Dict[str, torch.Tensor]] = {}
        for key, t in state.items():
            for part in ("lora_A", "lora_B"):
                if f".{part}." in key:
                    pairs.setdefault(key.split(f".{part}.")[0], {})[part] = t
        found = {}
        for name, layer in self.layers.items():
            hits = [m for m in pairs if m == name or m.endswith("." + name)]
            if len(hits) > 1 or (hits and len(pairs[hits[0]]) != 2):
                raise ValueError(f"adapter state: {name} has no single pair of lora_A and lora_B")
            if hits:
                a, b = pairs[hits[0]]["lora_A"], pairs[hits[0]]["lora_B"]
                r = a.shape[0]
                if r > layer.rank or a.shape != (r, layer.in_features) or b.shape != (layer.out_features, r):
                    raise ValueError(f"adapter state: {name} has shapes {tuple(a.shape)}, {tuple(b.shape)}")
                found[name] = (a, b)
        if not found:
            raise ValueError("adapter state: no key names a wrapped projection")
        for name, layer in self.layers.items():
            if name in found:
                a, b = found[name]
                layer.load(slot, a, b, alpha / a.shape[0])
            else:
                layer.unload(slot)
        return len(found)

    def unload(self, slot: int) -> None:
        for layer in self.layers.values():
            layer.unload(slot)

    def route(self, adapter: Optional[torch.Tensor], q_start: Optional[torch.Tensor] = None,
              tokens: Optional[int] = None) -> None:
        """adapter int32 [batch] slots on the model's device (-1: none), or None: no adapters.  The
        passes that follow are over [batch, T, hidden] or, with q_start int32 [batch + 1], over
        ``tokens`` packed rows; others are refused.  tokens None: as many as q_start[batch] says,
        which is read from the device (but not while a graph is captured: nothing is compared then)."""
        if adapter is not None and (adapter.dtype != torch.int32 or adapter.dim() != 1):
            raise ValueError("route: adapter must be int32 [batch]")
        if q_start is not None and (adapter is None or q_start.dtype != torch.int32 or q_start.shape != (adapter.shape[0] + 1,)):
            raise ValueError("route: q_start must be int32 [batch + 1] beside adapter [batch]")
        if tokens is not None and (q_start is None or tokens < 0):
            raise ValueError("route: tokens counts the rows of packed passes (with q_start)")
        if q_start is not None and tokens is None and not (q_start.is_cuda and torch.cuda.is_current_stream_capturing()):
            tokens = int(q_start[-1])
        self.routing.adapter, self.routing.q_start, self.routing.tokens = adapter, q_start, tokens
