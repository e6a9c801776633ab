"""Final norm + lm_head + cross-entropy on the device, forward and backward.

FitLLM seeds the backward of each micro-batch from its lm_head loss
(fitllm/backward.py:188-198): h_last -> final RMSNorm -> lm_head (bf16,
vocab 152,064, no bias) -> CrossEntropyLoss (mean over labels != -100) ->
(loss * loss_scale).backward() gives grad_h; the logged loss is the same mean
(fitllm/trainer.py:506-522, there on fp32 logits moved to the CPU).

Here, per micro-batch: RMSNorm (fitq_rmsnorm_fwd) -> logits = x.W^T on the
tcgen05 GEMM (bf16 [S, V]) -> fitq_cross_entropy turns the logits in place
into d(loss_scale * loss)/dlogits and writes the mean loss to a device scalar
-> dx = dlogits.W on the same GEMM (against Wᵀ, materialised once: the
lm_head is frozen) -> fitq_rmsnorm_bwd.  Nothing leaves the device and no
per-micro-batch synchronisation is needed; the losses stay on the device
until the caller reads them.
"""
from __future__ import annotations

from typing import List, NamedTuple, Optional, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib, ops


_LOGIT_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16,
                 torch.float32: _lib.DTYPE_F32}


class TokenLogProbs(NamedTuple):
    """logp and entropy fp32 [...], top_logp fp32 and top_ids int64 [..., top]."""
    logp: torch.Tensor
    entropy: torch.Tensor
    top_logp: torch.Tensor
    top_ids: torch.Tensor


def _row_stride(t: torch.Tensor) -> int:
    """Elements from row to row of [rows, V] (V where there is one row)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _logprobs_forward(logits, ids, top: int, want_stats: bool):
    """(logp, entropy, top_logp, top_ids, stats) of logits [rows, V] (fitq_token_logprobs)."""
    L = _lib.load()
    dev = logits.device
    rows, vocab = logits.shape
    logp = torch.empty(rows, dtype=torch.float32, device=dev)
    entropy = torch.empty_like(logp)
    stats = torch.empty(rows, 2, dtype=torch.float32, device=dev) if want_stats else None
    top_logp = torch.empty(rows, top, dtype=torch.float32, device=dev)
    top_ids = torch.empty(rows, top, dtype=torch.int64, device=dev)
    with ops._on(dev):
        _lib.check(L.fitq_token_logprobs(logits.data_ptr(), _LOGIT_DTYPES[logits.dtype], ids.data_ptr(), rows,
                                         vocab, _row_stride(logits), top, logp.data_ptr(), entropy.data_ptr(),
                                         _lib.ptr(stats), top_logp.data_ptr(), top_ids.data_ptr(),
                                         ops._raw_stream(dev.index)), "fitq_token_logprobs")
    return logp, entropy, top_logp, top_ids, stats


class _TokenLogProbsFn(torch.autograd.Function):
    """fitq_token_logprobs / fitq_token_logprobs_bwd over logits [rows, V]."""

    @staticmethod
    def forward(ctx, logits, ids, top: int):
        logp, entropy, top_logp, top_ids, stats = _logprobs_forward(logits, ids, top, True)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(top_ids)
        ctx.save_for_backward(logits, ids, stats, entropy, top_ids)
        return logp, entropy, top_logp, top_ids

    @staticmethod
    @once_differentiable
    def backward(ctx, g_logp, g_entropy, g_top, _):
        logits, ids, stats, entropy, top_ids = ctx.saved_tensors
        L = _lib.load()
        dev = logits.device
        rows, vocab = logits.shape
        top = top_ids.shape[1]
        g_logp, g_entropy, g_top = (None if g is None else g.contiguous() for g in (g_logp, g_entropy, g_top))
        d = torch.empty(rows, vocab, dtype=logits.dtype, device=dev)
        with ops._on(dev):
            _lib.check(L.fitq_token_logprobs_bwd(logits.data_ptr(), _LOGIT_DTYPES[logits.dtype], ids.data_ptr(),
                                                 rows, vocab, _row_stride(logits), top, stats.data_ptr(),
                                                 entropy.data_ptr(), top_ids.data_ptr(), _lib.ptr(g_logp),
                                                 _lib.ptr(g_entropy), _lib.ptr(g_top if top else None),
                                                 d.data_ptr(), ops._raw_stream(dev.index)), "fitq_token_logprobs_bwd")
        return d, None, None


def token_logprobs(logits: torch.Tensor, ids: torch.Tensor, top: int = 0) -> TokenLogProbs:
    """Log probabilities of given tokens, the rows' entropies and the `top` most
    likely tokens, in one read of the logits; differentiable (logp, entropy and
    top_logp) with one more read and one write.

    logits [..., V] bf16, fp16 or fp32 (rows may be strided, as in
    logits[..., :tokens]); ids [...] integers, an id outside [0, V) (-100 for
    instance) has logp 0 and no gradient.  Equal logits rank by index.  There is no
    forward-mode derivative."""
    if logits.dim() < 1 or ids.shape != logits.shape[:-1]:
        raise ValueError(f"token_logprobs: logits {tuple(logits.shape)} and ids {tuple(ids.shape)} do not match")
    if logits.dtype not in _LOGIT_DTYPES or not logits.is_cuda:
        raise ValueError("token_logprobs: logits must be a bf16, fp16 or fp32 CUDA tensor")
    if ids.device != logits.device or ids.dtype.is_floating_point or ids.dtype == torch.bool:
        raise ValueError("token_logprobs: ids must be integers on the logits' device")
    vocab = logits.shape[-1]
    if not 0 <= top <= min(64, vocab):
        raise ValueError(f"token_logprobs: top must be in 0..64 and at most {vocab} (got {top})")
    z = logits.reshape(-1, vocab) if logits.dim() != 2 else logits
    if (vocab > 1 and z.stride(1) != 1) or (z.shape[0] > 1 and z.stride(0) < vocab):
        z = z.contiguous()
    lead = ids.shape
    if len(lead) != 1 or ids.dtype != torch.int64 or not ids.is_contiguous():
        ids = ids.reshape(-1).to(torch.int64).contiguous()
    if forward_ad.unpack_dual(z).tangent is not None:  # the kernels would lose it
        raise NotImplementedError("token_logprobs: logits with a tangent (there is no forward-mode derivative)")
    if z.requires_grad and torch.is_grad_enabled():
        r = _TokenLogProbsFn.apply(z, ids, int(top))
    else:
        r = _logprobs_forward(z, ids, int(top), False)[:4]
    if len(lead) == 1:
        return TokenLogProbs(*r)
    return TokenLogProbs(r[0].view(lead), r[1].view(lead), r[2].view(*lead, top), r[3].view(*lead, top))


class LMHeadLoss:
    """Frozen final norm + lm_head with the reference's loss.

    norm_weight: [H] bf16; weight: [V, H] bf16 (nn.Linear layout)."""

    def __init__(self, norm_weight: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
                 ignore_index: int = -100):
        if weight.dtype != torch.bfloat16 or norm_weight.dtype != torch.bfloat16:
            raise TypeError("LMHeadLoss: bf16 norm weight and lm_head weight expected")
        self.norm_weight = norm_weight.contiguous()
        self.weight = weight.contiguous()
        self.weight_t = self.weight.t().contiguous()  # [H, V] for dx = dlogits . W
        self.eps = float(eps)
        self.ignore_index = int(ignore_index)

    @property
    def vocab(self) -> int:
        return int(self.weight.shape[0])

    def _norm(self, h2: torch.Tensor) -> torch.Tensor:
        L = _lib.load()
        y = torch.empty_like(h2)
        _lib.check(L.fitq_rmsnorm_fwd(h2.data_ptr(), self.norm_weight.data_ptr(), y.data_ptr(),
                                      h2.shape[0], h2.shape[1], self.eps, ops._stream(h2.device)),
                   "fitq_rmsnorm_fwd")
        return y

    def _norm_bwd(self, dy: torch.Tensor, h2: torch.Tensor) -> torch.Tensor:
        L = _lib.load()
        dx = torch.empty_like(h2)
        _lib.check(L.fitq_rmsnorm_bwd(dy.data_ptr(), h2.data_ptr(), self.norm_weight.data_ptr(),
                                      dx.data_ptr(), h2.shape[0], h2.shape[1], self.eps,
                                      ops._stream(h2.device)), "fitq_rmsnorm_bwd")
        return dx

    def logits(self, h: torch.Tensor) -> torch.Tensor:
        """[..., V] bf16 logits of the final hidden states (forward only)."""
        h2 = h.reshape(-1, h.shape[-1]).contiguous()
        return ops.gemm_bf16_tn(self._norm(h2), self.weight).view(*h.shape[:-1], self.vocab)

    def token_logprobs(self, h: torch.Tensor, ids: torch.Tensor, top: int = 0) -> TokenLogProbs:
        """token_logprobs of the lm_head logits of h [..., H] bf16 for ids [...],
        differentiable with respect to h (the head is frozen): policy or preference
        losses on log probabilities instead of the mean cross-entropy."""
        return token_logprobs(_LogitsFn.apply(h, self), ids, top)

    def loss_and_grad(self, h: torch.Tensor, labels: torch.Tensor,
                      loss_scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
        """One micro-batch: h [B, S, H] bf16 (last layer output), labels [B, S]
        int64 (already shifted, -100 ignored).  Returns (mean CE loss as a
        device fp32 scalar, grad of loss * loss_scale w.r.t. h, bf16)."""
        L = _lib.load()
        dev = h.device
        h2 = h.reshape(-1, h.shape[-1]).contiguous()
        rows = h2.shape[0]
        lab = labels.reshape(-1).to(device=dev, dtype=torch.int64).contiguous()
        if lab.numel() != rows:
            raise ValueError("loss_and_grad: labels must have one entry per token")
        with torch.cuda.device(dev):
            x = self._norm(h2)
            logits = ops.gemm_bf16_tn(x, self.weight)
            del x
            loss = torch.empty((), dtype=torch.float32, device=dev)
            nbytes = L.fitq_cross_entropy_workspace(rows)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            _lib.check(L.fitq_cross_entropy(logits.data_ptr(), lab.data_ptr(), rows, self.vocab,
                                            self.ignore_index, float(loss_scale), loss.data_ptr(),
                                            ws.data_ptr(), nbytes, ops._stream(dev)),
                       "fitq_cross_entropy")
            dx = ops.gemm_bf16_tn(logits, self.weight_t)  # logits now hold dlogits
            del logits
            grad = self._norm_bwd(dx, h2)
        return loss, grad.view_as(h)

    def loss_and_grad_microbatches(self, h: torch.Tensor, labels: torch.Tensor,
                                   loss_scale: float) -> Tuple[List[torch.Tensor], torch.Tensor]:
        """h [nmb, S, H], labels [nmb, S]: the reference's per-micro-batch loop
        (each micro-batch its own mean).  Returns (losses, grad_h [nmb, S, H])."""
        grad = torch.empty_like(h)
        losses = []
        for i in range(h.shape[0]):
            loss, g = self.loss_and_grad(h[i:i + 1], labels[i:i + 1], loss_scale)
            grad[i:i + 1] = g
            losses.append(loss)
        return losses, grad


class _LogitsFn(torch.autograd.Function):
    """LMHeadLoss.logits with the gradient with respect to h."""

    @staticmethod
    def forward(ctx, h, head: LMHeadLoss):
        h2 = h.reshape(-1, h.shape[-1]).contiguous()
        ctx.head = head
        ctx.save_for_backward(h2)
        with torch.cuda.device(h.device):
            return ops.gemm_bf16_tn(head._norm(h2), head.weight).view(*h.shape[:-1], head.vocab)

    @staticmethod
    @once_differentiable
    def backward(ctx, d):
        h2, = ctx.saved_tensors
        head = ctx.head
        with torch.cuda.device(d.device):
            dx = ops.gemm_bf16_tn(d.reshape(-1, head.vocab), head.weight_t)
            return head._norm_bwd(dx, h2).view(*d.shape[:-1], h2.shape[-1]), None


def random_lm_head(hidden: int, vocab: int, device, seed: int = 0, std: float = 0.02,
                   eps: float = 1e-6) -> LMHeadLoss:
    """Seeded N(0, std) bf16 lm_head with a unit final norm (synthetic workloads)."""
    g = torch.Generator(device=device).manual_seed(seed)
    w = (torch.randn(vocab, hidden, generator=g, device=device) * std).bfloat16()
    return LMHeadLoss(torch.ones(hidden, dtype=torch.bfloat16, device=device), w, eps=eps)
