"""The MoE router over many tokens, with its gradient, and its balance loss.

`route` is decode_step.route_tokens after the router's fp32 linear, as one kernel that also counts the tokens of every
expert: the same experts and weights, in decreasing order of choice, ties to the lower id. Its weights carry a
gradient to the logits (the choice itself has none; `bias` gets none, it is moved by the counts). `balance_loss` is the
auxiliary loss that keeps the experts evenly loaded, with its gradient. Both take CUDA tensors only.
"""
import functools

import torch

import _qmoe_lib as C
from dense_q import _on

MAX_EXPERTS = 1024
MAX_TOP_K = 32
_SCORES = {"sigmoid": 0, "softmax": 1}


def _logits(x, score):
    if score not in _SCORES:
        raise C.QmoeError(f"score is 'sigmoid' or 'softmax' (got {score!r})")
    if x.dim() != 2 or not 1 <= x.shape[1] <= MAX_EXPERTS:
        raise C.QmoeError(f"logits must be [T, E] with 1 <= E <= {MAX_EXPERTS} (got {tuple(x.shape)})")
    C.dtype_code(x)
    C.ptr(x)


def _rows(x):
    """x with unit column stride and rows that do not overlap, and its row stride."""
    if x.is_contiguous():
        return x, x.shape[1]
    if x.stride(1) != 1 or (x.shape[0] > 1 and x.stride(0) < x.shape[1]):
        x = x.contiguous()
    return x, int(x.stride(0)) if x.shape[0] > 1 else x.shape[1]


def _route(x, bias, top_k, scaling, n_group, topk_group, norm, score):
    x, ld = _rows(x)
    T, E = x.shape
    dev = x.device
    ids = torch.empty(T, top_k, dtype=torch.int64, device=dev)
    w = torch.empty(T, top_k, dtype=torch.float32, device=dev)
    counts = torch.empty(E, dtype=torch.int32, device=dev) if T else torch.zeros(E, dtype=torch.int32, device=dev)
    if T:
        with _on(x):
            C.call("qmoe_route", x.data_ptr(), C.DT[x.dtype], ld, bias.data_ptr() if bias is not None else None, T, E, top_k,
                   n_group, topk_group, norm, score, scaling, ids.data_ptr(), w.data_ptr(), counts.data_ptr(), C.stream_of(x))
    return ids, w, counts


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, *args):
        ids, w, counts = _route(logits, *args)
        ctx.save_for_backward(logits, ids)
        ctx.args = args[1:]
        ctx.mark_non_differentiable(ids, counts)
        ctx.set_materialize_grads(False)
        return ids, w, counts

    @staticmethod
    def backward(ctx, *grads):
        return (_Route.twice if torch.is_grad_enabled() else _Route.once)(ctx, *grads)

    @staticmethod
    def once(ctx, _ids, dw, _counts):
        if dw is None:
            return (None,) * 8
        logits, ids = ctx.saved_tensors
        top_k, scaling, _, _, norm, score = ctx.args
        x, ld = _rows(logits)
        dl = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        if x.shape[0]:
            dw = dw.to(torch.float32).contiguous()
            with _on(x):
                C.call("qmoe_route_backward", x.data_ptr(), C.DT[x.dtype], ld, x.shape[0], x.shape[1], top_k, norm, score, scaling,
                       ids.data_ptr(), C.ptr(dw), dl.data_ptr(), C.stream_of(x))
        return dl, None, None, None, None, None, None, None

    twice = staticmethod(torch.autograd.function.once_differentiable(once.__func__))   # of a graph: refuses a second


def route(logits, bias=None, top_k=22, scaling=5.0, n_group=1, topk_group=1, norm_topk_prob=False, score="sigmoid"):
    """logits [T, E] (fp32, bf16 or fp16; E <= 1024) -> ids int64 [T, top_k], weights f32 [T, top_k], counts int32 [E].
    Score sigmoid(logit), choice score + bias [E] f32; with n_group > 1 only the topk_group groups whose two best
    choices have the largest sum keep theirs (the others' become 0, as the model's router has it); the top_k <= 32
    largest choices; weight = score, divided by the sum of the chosen (+ 1e-20) with norm_topk_prob, times scaling.
    score "softmax": the softmax over the experts, chosen by the logits, no bias, groups left out entirely. A NaN is
    chosen last. Differentiable in the logits through the weights."""
    _logits(logits, score)
    T, E = logits.shape
    if not 1 <= top_k <= min(MAX_TOP_K, E):
        raise C.QmoeError(f"top_k must lie in 1..{min(MAX_TOP_K, E)} (got {top_k})")
    if not 1 <= n_group <= 32 or E % n_group or not 1 <= topk_group <= n_group or (n_group > 1 and E // n_group < 2):
        raise C.QmoeError(f"{E} experts do not split into {n_group} groups of two or more, {topk_group} of them kept")
    if bias is not None:
        if score == "softmax":
            raise C.QmoeError("a softmax router takes no bias")
        if bias.shape != (E,) or bias.device != logits.device:
            raise C.QmoeError("bias must be [E], on the logits' device")
        bias = bias.detach().to(torch.float32).contiguous()
    args = (bias, int(top_k), float(scaling), int(n_group), int(topk_group), int(bool(norm_topk_prob)), _SCORES[score])
    if logits.requires_grad and torch.is_grad_enabled():
        return _Route.apply(logits, *args)
    return _route(logits, *args)


_bytes = functools.lru_cache(maxsize=256)(lambda T, E: int(C.lib().qmoe_balance_workspace_bytes(T, E)))


def _balance(x, ids, mask, score, coef):
    """Loss, counts, and coef * f / T' per expert for the backward pass."""
    x, ld = _rows(x)
    T, E = x.shape
    dev = x.device
    if T == 0:
        return torch.zeros((), device=dev), torch.zeros(E, dtype=torch.int32, device=dev), torch.zeros(E, device=dev)
    loss, counts = torch.empty((), dtype=torch.float32, device=dev), torch.empty(E, dtype=torch.int32, device=dev)
    c = torch.empty(E, dtype=torch.float32, device=dev)
    n = _bytes(T, E)
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    with _on(x):
        C.call("qmoe_balance", x.data_ptr(), C.DT[x.dtype], ld, ids.data_ptr(), int(ids.dtype == torch.int64),
               mask.data_ptr() if mask is not None else None, T, E, ids.shape[1], score, coef, loss.data_ptr(), counts.data_ptr(),
               c.data_ptr(), ws.data_ptr(), n, C.stream_of(x))
    return loss, counts, c


class _Balance(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, mask, score, coef):
        loss, counts, c = _balance(logits, ids, mask, score, coef)
        ctx.save_for_backward(logits, mask, c)
        ctx.score = score
        ctx.mark_non_differentiable(counts)
        ctx.set_materialize_grads(False)
        return loss, counts

    @staticmethod
    def backward(ctx, *grads):
        return (_Balance.twice if torch.is_grad_enabled() else _Balance.once)(ctx, *grads)

    @staticmethod
    def once(ctx, dloss, _counts):
        if dloss is None:
            return (None,) * 5
        logits, mask, c = ctx.saved_tensors
        x, ld = _rows(logits)
        dl = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        if x.shape[0]:
            g = dloss.to(torch.float32)
            with _on(x):
                C.call("qmoe_balance_backward", x.data_ptr(), C.DT[x.dtype], ld, mask.data_ptr() if mask is not None else None,
                       x.shape[0], x.shape[1], ctx.score, c.data_ptr(), C.ptr(g), dl.data_ptr(), C.stream_of(x))
        return dl, None, None, None, None

    twice = staticmethod(torch.autograd.function.once_differentiable(once.__func__))


def balance_loss(logits, ids, mask=None, score="sigmoid", coef=1.0):
    """logits [T, E] (fp32, bf16 or fp16), ids [T, k] int64 or int32 (of route) -> (loss f32 [], counts int32 [E]):
    loss = coef * sum_e f_e P_e with f_e = E * counts_e / (k * T') and P_e the mean over tokens of score_e / sum of the
    token's scores; 1 * coef when the experts are evenly loaded. mask [T] bool: tokens with False (padding) count
    nowhere, T' are the others; none left: loss 0. Ids outside [0, E) are not counted. Differentiable in the logits
    (f is held fixed, as the counts have no gradient). Sums run in a fixed order."""
    _logits(logits, score)
    T = logits.shape[0]
    if ids.dim() != 2 or ids.shape[0] != T or ids.shape[1] < 1 or ids.dtype not in (torch.int64, torch.int32):
        raise C.QmoeError("ids must be int64 or int32 [T, k] with k >= 1")
    if ids.device != logits.device:
        raise C.QmoeError("ids must be on the logits' device")
    if mask is not None:
        if mask.shape != (T,) or mask.dtype != torch.bool or mask.device != logits.device:
            raise C.QmoeError("mask must be bool [T], on the logits' device")
        mask = mask.contiguous()
    args = (ids.contiguous(), mask, _SCORES[score], float(coef))
    if logits.requires_grad and torch.is_grad_enabled():
        return _Balance.apply(logits, *args)
    return _balance(logits, *args)[:2]
