"""The MoE router over many tokens, with its gradient, and its balance loss.

`route` is decode_step.route_tokens after the router's fp32 linear, as one kernel that also counts the tokens of every
expert: the same experts and weights, in decreasing order of choice, ties to the lower id. Its weights carry a
gradient to the logits (the choice itself has none; `bias` gets none, it is moved by the counts). `balance_loss` is the
auxiliary loss that keeps the experts evenly loaded, with its gradient. Both take CUDA tensors only.
"""
import _qmoe_lib as C


def route(logits, bias=None, top_k=22, scaling=5.0, n_group=1, topk_group=1, norm_topk_prob=False, score="sigmoid"):
    """logits [T, E] (fp32, bf16 or fp16; E <= 1024) -> ids int64 [T, top_k], weights f32 [T, top_k], counts int32 [E].
    Score sigmoid(logit), choice score + bias [E] f32; with n_group > 1 only the topk_group groups whose two best
    choices have the largest sum keep theirs (the others' become 0, as the model's router has it); the top_k <= 32
    largest choices; weight = score, divided by the sum of the chosen (+ 1e-20) with norm_topk_prob, times scaling.
    score "softmax": the softmax over the experts, the choice is the logit, no bias; groups are ranked by the sum of their
    two best logits (the order of the product of their two best scores, which is not that of the scores' sum or of the
    best score alone) and left out entirely, so the kept ones need top_k experts, and one of them with a logit of -inf
    is chosen before any that is left out. A NaN counts as -inf. Differentiable in the logits through the weights."""
    return C.bind().route(logits, bias, top_k, scaling, n_group, topk_group, norm_topk_prob, score)


def balance_loss(logits, ids, mask=None, score="sigmoid", coef=1.0):
    """logits [T, E] (fp32, bf16 or fp16), ids [T, k] int64 or int32 (of route) -> (loss f32 [], counts int32 [E]):
    loss = coef * sum_e f_e P_e with f_e = E * counts_e / (k * T') and P_e the mean over tokens of score_e / sum of the
    token's scores; 1 * coef when the experts are evenly loaded. mask [T] bool: tokens with False (padding) count
    nowhere, T' are the others; none left: loss 0. Ids outside [0, E) are not counted, one that is twice in a row counts twice. Differentiable in the logits
    (f is held fixed, as the counts have no gradient). Sums run in a fixed order."""
    return C.bind().balance_loss(logits, ids, mask, score, coef)
