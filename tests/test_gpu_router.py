"""The router over many tokens and its balance loss (router.route / balance_loss).

Chosen experts have to equal those of torch's fp32 scores sorted stably (ties to the lower id). Weights, losses and
gradients are compared with 64-bit formulas: a sigmoid or a softmax term in fp32 is off by a few units of 2^-24 (exp 1
last place, two roundings more), sums of n positive terms by n 2^-24 at most and far less in a tree; 2^-18 relative to the
quantities that are subtracted covers them with room for sums of 1024 experts or 4096 tokens."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
TOL = 2.0 ** -18


def seeded(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def chosen(logits, bias, k, n_group=1, topk_group=1, score="sigmoid"):
    x = logits.float()
    c = torch.sigmoid(x) if score == "sigmoid" else x
    if bias is not None:
        c = c + bias
    c = torch.where(torch.isnan(c), -float("inf"), c)
    if n_group > 1:
        g = c.view(c.shape[0], n_group, -1)
        best = torch.sort(g, dim=-1, descending=True)[0][..., :2].sum(-1)
        keep = torch.zeros_like(best, dtype=torch.bool)
        keep.scatter_(1, torch.sort(best, dim=-1, descending=True, stable=True)[1][:, :topk_group], True)
        c = torch.where(keep[..., None], g, 0.0 if score == "sigmoid" else -float("inf")).reshape(c.shape)
    return torch.sort(c, dim=-1, descending=True, stable=True)[1][:, :k]


def weights64(x, ids, scaling, norm, score):
    s = torch.sigmoid(x) if score == "sigmoid" else torch.softmax(x, -1)
    w = s.gather(1, ids)
    return (w / (w.sum(-1, keepdim=True) + 1e-20) if norm else w) * scaling


def check_route(logits, bias, k, score="sigmoid", norm=False, groups=(1, 1), scaling=5.0, grad=True):
    import router as R
    leaf = logits.detach().clone(memory_format=torch.preserve_format).requires_grad_()
    ids, w, n = R.route(leaf, bias, top_k=k, scaling=scaling, n_group=groups[0], topk_group=groups[1], norm_topk_prob=norm,
                        score=score)
    T, E = logits.shape
    assert ids.dtype == torch.int64 and n.dtype == torch.int32 and w.dtype == torch.float32
    assert torch.equal(ids, chosen(logits, bias, k, *groups, score))
    assert torch.equal(n, torch.bincount(ids.flatten(), minlength=E).to(torch.int32))
    x = logits.double().requires_grad_()
    ref = weights64(x, ids, scaling, norm, score)
    assert torch.allclose(w.double(), ref, rtol=TOL, atol=scaling * 1e-30)
    if not grad:
        return
    dw = torch.randn(T, k, generator=seeded(T + E), device=DEV)
    got, = torch.autograd.grad(w, leaf, dw)
    want, = torch.autograd.grad(ref, x, dw.double())
    assert got.dtype == logits.dtype and got.shape == logits.shape
    # what the gradient subtracts: |dw| s sums to at most scaling * sum |dw| * max score
    size = scaling * dw.abs().double().sum(-1, keepdim=True) * ref.abs().amax(-1, keepdim=True) / scaling + 1e-30
    if norm:
        size = scaling * dw.abs().double().sum(-1, keepdim=True)
    half = torch.finfo(logits.dtype).eps / 2
    tiny = torch.finfo(logits.dtype).smallest_normal * torch.finfo(logits.dtype).eps
    assert bool(((got.double() - want).abs() <= TOL * size + half * want.abs() + tiny).all())


CASES = [(1, 512, 22), (1, 1, 1), (2, 7, 7), (9, 33, 5), (64, 512, 22), (131, 128, 6), (1000, 1024, 32), (5000, 512, 22), (77, 60, 8),
         (40, 257, 17), (3, 1000, 1)]


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("T,E,k", CASES)
def test_route(T, E, k, score, norm):
    g = seeded(T * E + k)
    x = torch.randn(T, E, generator=g, device=DEV) * 2 - 1
    bias = torch.randn(E, generator=g, device=DEV) * 0.01 if score == "sigmoid" else None
    check_route(x, bias, k, score, norm)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_route_of_short_types(dtype, score):
    """Many equal logits in a row: equal choices go to the lower expert."""
    x = (torch.randn(300, 200, generator=seeded(3), device=DEV) * 2).to(dtype)
    check_route(x, None, 12, score)
    check_route(x, None, 12, score, norm=True)


@pytest.mark.parametrize("groups", [(8, 4), (4, 2), (2, 1), (32, 3)])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_route_in_groups(groups, score):
    g = seeded(groups[0])
    for E in (64, 512, 960):
        x = torch.randn(50, E, generator=g, device=DEV)
        bias = torch.randn(E, generator=g, device=DEV) * 0.2 if score == "sigmoid" else None   # some choices below 0
        check_route(x, bias, min(22, E * groups[1] // groups[0]), score, True, groups)


def test_route_ties_and_strange_numbers():
    E = 96
    x = torch.zeros(12, E, device=DEV)
    x[1, 40:] = 1.0
    x[2] = -200.0                                          # scores of 0
    x[3] = 200.0                                           # scores of 1
    x[4, ::2] = -float("inf")
    x[5, 10], x[5, 90] = float("inf"), -float("inf")
    x[6, 3:60] = float("nan")
    x[7] = torch.arange(E, device=DEV) % 3
    x[8] = -0.0
    x[8, 50:] = 0.0
    x[9] = float("nan")
    x[10] = -torch.arange(E, device=DEV).float()
    x[11] = 20.0 + torch.arange(E, device=DEV) * 0.1       # scores that differ in the last places, or not at all
    import router as R
    for bias in (None, torch.zeros(E, device=DEV), torch.linspace(-1, 1, E, device=DEV)):
        for k in (1, 22, 32):
            ids, w, n = R.route(x, bias, top_k=k)
            assert torch.equal(ids, chosen(x, bias, k))
            assert torch.equal(n, torch.bincount(ids.flatten(), minlength=E).to(torch.int32))
            assert torch.equal(w, torch.sigmoid(x).gather(1, ids) * 5.0) or torch.isnan(w).any()
    ids, _, _ = R.route(x[:9], None, top_k=22, score="softmax")
    assert torch.equal(ids, chosen(x[:9], None, 22, score="softmax"))


def test_route_equals_the_torch_router():
    """The framework's torch router on the same logits: the same experts, bit-identical weights."""
    import decode_step as DS
    import router as R
    g = seeded(21)
    x = torch.randn(2000, 256, generator=g, device=DEV)
    gate = torch.randn(512, 256, generator=g, device=DEV) * 0.05
    bias = torch.randn(512, generator=g, device=DEV) * 0.01
    ids, w = DS.route_tokens(x, gate, bias)
    logits = torch.nn.functional.linear(x, gate)
    got, gw, _ = R.route(logits, bias)
    o, p = ids.sort(-1), got.sort(-1)
    assert torch.equal(o[0], p[0]) and torch.equal(w.gather(1, o[1]), gw.gather(1, p[1]))


def test_sigmoid_is_torchs():
    """The choice is made on fp32 scores: over the whole range they are torch's own bits."""
    import router as R
    x = torch.linspace(-30, 30, 1 << 20, device=DEV).view(-1, 32)
    x = torch.cat([x, torch.randn(1 << 15, 32, generator=seeded(2), device=DEV)])
    ids, w, _ = R.route(x, None, top_k=32, scaling=1.0)
    assert torch.equal(w, torch.sigmoid(x).gather(1, ids))


def test_route_strides_streams_and_replay():
    import router as R
    g = seeded(12)
    big = torch.randn(128, 600, generator=g, device=DEV)
    for x in (big[:, 3:515], big[::2, :512], big.t()[:512, :100].t(), big[:1, 5:500], big[:0, :64]):
        if x.shape[0]:
            check_route(x, None, 9)
        else:
            ids, w, n = R.route(x, None, top_k=9)
            assert ids.shape == (0, 9) and not n.any()
    x = big[:, :512].contiguous()
    want = R.route(x, None)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = R.route(x, None)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    buf = x.clone()
    with torch.cuda.graph(graph):
        out = R.route(buf, None)
    for y in (x, big[:, 50:562].contiguous(), x):
        buf.copy_(y)
        graph.replay()
        graph.replay()                                     # counts start from zero in every replay
        assert all(torch.equal(a, b) for a, b in zip(out, R.route(y, None)))


# ------------------------------------------------------------------------------------------------ balance loss
def loss64(x, ids, mask, score, coef):
    T, E = x.shape
    keep = torch.ones(T, dtype=torch.bool, device=DEV) if mask is None else mask
    rows = int(keep.sum())
    i = ids[keep].long().flatten()
    i = i[(i >= 0) & (i < E)]
    n = torch.bincount(i, minlength=E)
    if rows == 0:
        return x.sum() * 0, n, torch.zeros(E, dtype=torch.float64, device=DEV)
    f = n.double() * E / (ids.shape[1] * rows)
    s = torch.sigmoid(x) if score == "sigmoid" else torch.softmax(x, -1)
    p = (s / s.sum(-1, keepdim=True))[keep]
    return coef * (f * p.mean(0)).sum(), n, coef * f / rows


def check_balance(logits, ids, mask=None, score="sigmoid", coef=1.0):
    """p from logarithms of the scores (log sigmoid(x) is x to 1e-13 below -30), so that none underflows, and the gradient
    by its formula p_j (c_j - sum c p) (1 - s_j); test_training_step_of_both_and_reruns has it by automatic
    differentiation, test_gradients_against_differences by differences."""
    import router as R
    leaf = logits.detach().clone().requires_grad_()
    loss, n = R.balance_loss(leaf, ids, mask, score, coef)
    got, = torch.autograd.grad(loss * 3.0, leaf)
    loss = loss.detach()
    x = logits.double()
    keep = torch.ones(x.shape[0], dtype=torch.bool, device=DEV) if mask is None else mask
    x = torch.where(keep[:, None], x, 0.0)                 # what masked rows hold does not matter
    ls = x if score == "softmax" else torch.where(x < -30, x, -torch.log1p(torch.exp(-x)))
    p = torch.where(keep[:, None], torch.exp(ls - torch.logsumexp(ls, -1, keepdim=True)), 0.0)
    rows = int(keep.sum())
    i = ids[keep].long().flatten()
    n64 = torch.bincount(i[(i >= 0) & (i < x.shape[1])], minlength=x.shape[1])
    f = n64.double() * x.shape[1] / (ids.shape[1] * max(rows, 1))
    c = coef * f / max(rows, 1)
    want = coef * (f * p.sum(0) / max(rows, 1)).sum()
    assert torch.equal(n, n64.to(torch.int32)) and loss.shape == () and loss.dtype == torch.float32
    assert abs(float(loss) - float(want)) <= TOL * abs(float(want))
    one_less = torch.sigmoid(-x) if score == "sigmoid" else 1.0
    ref = 3 * p * (c - (c * p).sum(-1, keepdim=True)) * one_less
    half = torch.finfo(logits.dtype).eps / 2
    tiny = torch.finfo(logits.dtype).smallest_normal * torch.finfo(logits.dtype).eps
    size = 3 * p * (c + (c * p).sum(-1, keepdim=True))     # the two terms that are subtracted
    assert got.dtype == logits.dtype
    # 2^-90: in a row whose largest logit is -20 or more, a score below e^-87 counts as e^-87: p under e^-67 (96 bits down)
    assert bool(((got.double() - ref).abs() <= TOL * size + half * ref.abs() + tiny + 2.0 ** -90 * (c + (c * p).sum(-1, keepdim=True))).all())
    assert not got[~keep].any()
    return loss, got


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 512, 22), (5, 7, 2), (64, 33, 32), (300, 128, 6), (1001, 512, 22), (4096, 1024, 8), (9, 257, 40)])
def test_balance(T, E, k, score, dtype):
    g = seeded(T + E)
    x = (torch.randn(T, E, generator=g, device=DEV) * 1.5).to(dtype)
    ids = torch.topk(x.float(), min(k, E), -1)[1]
    check_balance(x, ids, None, score, 0.01)
    mask = torch.rand(T, generator=g, device=DEV) < 0.6
    check_balance(x, ids.to(torch.int32), mask, score)


def test_balance_masks_and_odd_ids():
    g = seeded(31)
    x = torch.randn(50, 64, generator=g, device=DEV)
    ids = torch.randint(0, 64, (50, 5), generator=g, device=DEV)
    ids[3] = -1
    ids[4, 2] = 64
    ids[5] = 7                                             # the same expert five times
    mask = torch.zeros(50, dtype=torch.bool, device=DEV)
    loss, grad = check_balance(x, ids, mask)               # nothing left
    assert float(loss) == 0.0 and not grad.any()
    mask[17] = True
    check_balance(x, ids, mask)                            # one token
    mask[:40] = True
    y = x.clone()
    y[40:] = float("nan")
    y[45] = float("inf")
    y[46] = torch.finfo(torch.float32).min
    a, b = check_balance(y, ids, mask), check_balance(x, ids, mask)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    import router as R
    loss, n = R.balance_loss(x[:0], ids[:0])
    assert float(loss) == 0.0 and not n.any()


def test_balance_of_extreme_logits():
    """Rows so low that every sigmoid underflows keep their ratios; large logits, and an expert ruled out by -inf or the
    lowest number, have p = 0 there."""
    g = seeded(61)
    x = torch.randn(40, 96, generator=g, device=DEV)
    x[:8] -= 30
    x[8:16] -= 120
    x[16:24] -= 3000
    x[24:32] += 100
    ids = torch.topk(x, 4)[1]
    check_balance(x[:24], ids[:24])
    check_balance(x[24:], ids[24:])
    y = x[32:].clone()
    y[:, 5] = -float("inf")
    y[:, 7] = torch.finfo(torch.float32).min
    for score in ("sigmoid", "softmax"):
        _, grad = check_balance(y, ids[32:], None, score)
        assert float(grad[:, [5, 7]].abs().max()) < 1e-30


def test_second_gradients_are_refused():
    import router as R
    x = torch.randn(8, 16, generator=seeded(3), device=DEV, requires_grad=True)
    ids, w, _ = R.route(x, None, top_k=2)
    for out in (w.sum(), R.balance_loss(x, ids)[0]):
        first, = torch.autograd.grad(out, x, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(first.sum(), x)


def test_even_load_gives_one():
    import router as R
    ids = torch.arange(512, device=DEV).view(64, 8)
    loss, n = R.balance_loss(torch.zeros(64, 512, device=DEV), ids)
    assert abs(float(loss) - 1.0) <= TOL and bool((n == 1).all())


def test_gradients_against_differences():
    """Central differences of the forward passes' own values, in directions of random signs. With step h the fp32 values'
    error 2^-22 |L| / h and the third derivative's h^2 stay below 1 % of the directional derivative's scale."""
    import router as R
    g = seeded(41)
    x = torch.randn(16, 24, generator=g, device=DEV)
    dw = torch.randn(16, 4, generator=g, device=DEV)
    h = 2.0 ** -7
    for score in ("sigmoid", "softmax"):
        ids0, _, _ = R.route(x, None, top_k=4, score=score)

        def weights(y):
            return weights64(y.double(), ids0, 5.0, True, score)

        leaf = x.clone().requires_grad_()
        ids, w, _ = R.route(leaf, None, top_k=4, norm_topk_prob=True, score=score)
        grad = torch.autograd.grad(w, leaf, dw)[0]
        lossg = torch.autograd.grad(R.balance_loss(leaf, ids0, score=score)[0], leaf)[0]
        for seed in range(4):
            d = torch.sign(torch.randn(16, 24, generator=seeded(seed), device=DEV))
            num = ((weights(x + h * d) - weights(x - h * d)) * dw).sum() / (2 * h)
            assert abs(float(num) - float((grad.double() * d).sum())) <= 0.01 * float((grad.abs()).sum())
            up, down = (float(R.balance_loss(x + v * d, ids0, score=score)[0]) for v in (h, -h))
            assert abs((up - down) / (2 * h) - float((lossg.double() * d).sum())) <= 0.01 * float(lossg.abs().sum())


def test_training_step_of_both_and_reruns():
    """One step's gradient through the weights and the loss together, twice: the same bits; and as a captured graph."""
    import router as R
    g = seeded(51)
    x = torch.randn(700, 512, generator=g, device=DEV)
    dw = torch.randn(700, 22, generator=g, device=DEV)

    def step(v):
        leaf = v.detach().requires_grad_()
        ids, w, n = R.route(leaf, None, norm_topk_prob=True)
        loss, m = R.balance_loss(leaf, ids, coef=0.01)
        return torch.autograd.grad([w, loss], leaf, [dw, torch.ones_like(loss)])[0], n, m, loss.detach()

    a, b = step(x), step(x)
    assert all(torch.equal(u, v) for u, v in zip(a, b)) and torch.equal(a[1], a[2])
    y = x.double().requires_grad_()
    ids = chosen(x, None, 22)
    ref = torch.autograd.grad([weights64(y, ids, 5.0, True, "sigmoid"), loss64(y, ids, None, "sigmoid", 0.01)[0]], y,
                              [dw.double(), torch.ones((), dtype=torch.float64, device=DEV)])[0]
    assert bool(((a[0].double() - ref).abs() <= 2 * TOL * 5 * dw.abs().double().sum(-1, keepdim=True)).all())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x)
    torch.cuda.current_stream().wait_stream(side)
    buf = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(buf)
    for v in (x, x.flip(0)):
        buf.copy_(v)
        graph.replay()
        assert all(torch.equal(p, q) for p, q in zip(out, step(v)))


def test_only_what_is_asked_for_is_differentiated():
    import router as R
    x = torch.randn(8, 16, generator=seeded(1), device=DEV, requires_grad=True)
    ids, w, n = R.route(x, None, top_k=2)
    assert not ids.requires_grad and not n.requires_grad and w.requires_grad
    w.sum().backward()                                     # an expanded gradient
    assert x.grad is not None
    with torch.no_grad():
        assert not R.route(x, None, top_k=2)[1].requires_grad
    bias = torch.zeros(16, device=DEV, requires_grad=True)
    R.route(x, bias, top_k=2)[1].sum().backward()
    assert bias.grad is None


def test_groups_of_opposite_infinities():
    """A group whose two best choices are +inf and -inf has no sum: it comes last, and topk_group groups are kept."""
    import router as R
    bias = torch.zeros(8, device=DEV)
    bias[0], bias[1] = float("inf"), -float("inf")
    ids, _, _ = R.route(torch.zeros(3, 8, device=DEV), bias, top_k=8, n_group=4, topk_group=2)
    # groups 1 and 2 are kept with choices of 0.5, the others' become 0: ties to the lower id
    assert ids.tolist() == [[2, 3, 4, 5, 0, 1, 6, 7]] * 3


def test_ids_that_are_none_take_no_part_in_the_gradient():
    """The C entry with ids outside the experts (a caller's own list): as if they were not chosen."""
    import _qmoe_lib as C
    g = seeded(71)
    x = torch.randn(5, 40, generator=g, device=DEV)
    dw = torch.randn(5, 6, generator=g, device=DEV)
    ids = torch.topk(x, 6)[1]
    ids[:, 2] = torch.tensor([-1, 40, 1 << 40, -(1 << 40), 41], device=DEV)
    for score in (0, 1):
        for norm in (0, 1):
            dl = torch.empty_like(x)
            C.call("qmoe_route_backward", C.ptr(x), 0, 40, 5, 40, 6, norm, score, 5.0, C.ptr(ids), C.ptr(dw), C.ptr(dl), C.stream_of(x))
            y = x.double().requires_grad_()
            keep = [0, 1, 3, 4, 5]
            w = weights64(y, ids[:, keep], 5.0, norm == 1, ("sigmoid", "softmax")[score])
            ref = torch.autograd.grad(w, y, dw[:, keep].double())[0]
            assert bool(((dl.double() - ref).abs() <= TOL * 5 * dw.abs().double().sum(-1, keepdim=True)).all())


def test_route_refusals():
    import _qmoe_lib as C
    import router as R
    x = torch.zeros(4, 64, device=DEV)
    ids = torch.zeros(4, 2, dtype=torch.int64, device=DEV)
    for bad, word in ((lambda: R.route(x, score="softmax", top_k=17, n_group=8, topk_group=2), "leaves 16"),
                      (lambda: R.route(x, torch.zeros(64, device=DEV), score="softmax"), "no bias"),
                      (lambda: R.route(x, torch.zeros(63, device=DEV)), "bias must"), (lambda: R.route(x, top_k=33), "top_k"),
                      (lambda: R.route(x, n_group=5), "groups"), (lambda: R.balance_loss(x, ids[:3]), "ids must"),
                      (lambda: R.balance_loss(x, ids.float()), "ids must"), (lambda: R.balance_loss(x, ids.cpu()), "device"),
                      (lambda: R.balance_loss(x, ids, torch.ones(4, device=DEV)), "mask must")):
        with pytest.raises(C.QmoeError, match=word):
            bad()


@pytest.mark.parametrize("T", [1, 7, 8, 9, 63, 64, 65, 2959, 2960, 2961, 3500, 4737])
def test_route_counts_at_the_launch_borders(T):
    check_route(torch.randn(T, 96, generator=seeded(T), device=DEV), None, 6, grad=False)


def test_backward_into_a_graph():
    """loss.backward() captured after warm-up, both operators together, twice through a non-leaf; replayed on new inputs."""
    import router as R
    x = torch.randn(300, 64, generator=seeded(81), device=DEV, requires_grad=True)
    gate = torch.randn(128, 64, generator=seeded(82), device=DEV, requires_grad=True)

    def step():
        ids, w, _ = R.route(x @ gate.t(), None, top_k=4, norm_topk_prob=True)
        (R.balance_loss(x @ gate.t(), ids, coef=0.1)[0] + w.square().sum()).backward()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    x.grad.zero_(), gate.grad.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for seed in (83, 84):
        with torch.no_grad():
            x.copy_(torch.randn(300, 64, generator=seeded(seed), device=DEV))
        x.grad.zero_(), gate.grad.zero_()
        graph.replay()
        got = x.grad.clone(), gate.grad.clone()
        x.grad.zero_(), gate.grad.zero_()
        step()
        for a, b in zip(got, (x.grad, gate.grad)):
            assert torch.allclose(a, b, rtol=1e-5, atol=1e-5 * float(b.abs().max()))


@pytest.mark.parametrize("E", [96, 512, 1000])
@pytest.mark.parametrize("T", [1, 16, 17, 31, 33, 255, 256, 257, 511, 512, 513])
def test_balance_at_the_launch_borders(T, E):
    """One CTA, a cluster with ragged parts, and the two kernels: loss, counts and gradient, masked and not."""
    g = seeded(T + E)
    x = torch.randn(T, E, generator=g, device=DEV)
    ids = torch.randint(0, E, (T, 5), generator=g, device=DEV)
    for mask in (None, torch.rand(T, generator=g, device=DEV) < 0.6):
        for score in ("sigmoid", "softmax"):
            check_balance(x, ids, mask, score, 0.5)


def test_graphs_that_are_used_twice_or_changed():
    import _qmoe_lib as C
    import router as R
    import torch.autograd.forward_ad as fwd
    x = torch.randn(20, 32, generator=seeded(61), device=DEV, requires_grad=True)
    for f in (lambda v: R.route(v, None, top_k=3)[1].square().sum(),
              lambda v: R.balance_loss(v, torch.topk(v.detach(), 3)[1], torch.ones(20, dtype=torch.bool, device=DEV))[0]):
        out = f(x)
        a, = torch.autograd.grad(out, x, retain_graph=True)
        b, = torch.autograd.grad(out, x)
        assert torch.equal(a, b)
        with pytest.raises(RuntimeError, match="second time"):
            torch.autograd.grad(out, x)
        y = x * 1.0
        out = f(y)
        y.mul_(2.0)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            torch.autograd.grad(out, x)
        with fwd.dual_level(), pytest.raises(C.QmoeError, match="forward-mode"):
            f(fwd.make_dual(x.detach(), torch.ones_like(x)))
    ids, w, _ = R.route(x, None, top_k=3)
    ids.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(w.sum(), x)


def test_gradients_of_views_and_copies():
    """Logits that are views, broadcast over tokens or strided: the gradient has their shape, and sums where they share."""
    import router as R
    g = seeded(62)
    row = torch.randn(1, 48, generator=g, device=DEV, requires_grad=True)
    wide = torch.randn(30, 96, generator=g, device=DEV, requires_grad=True)
    ids = torch.randint(0, 48, (30, 4), generator=g, device=DEV)
    for leaf, view in ((row, lambda v: v.expand(30, 48)), (wide, lambda v: v[:, 3:51]), (wide, lambda v: v[:, ::2]), (wide, lambda v: v.t()[:30, :30])):
        def both(z, make):
            n = z.shape[1]
            i = ids % n
            return make(z, i)
        got, = torch.autograd.grad(both(view(leaf), lambda z, i: R.balance_loss(z, i)[0]), leaf)
        y = leaf.detach().double().requires_grad_()
        want, = torch.autograd.grad(both(view(y), lambda z, i: loss64(z, i, None, "sigmoid", 1.0)[0]), y)
        assert got.shape == leaf.shape and bool(((got.double() - want).abs() <= 4 * TOL * want.abs().max()).all())
        dw = torch.randn(view(leaf).shape[0], 4, generator=seeded(5), device=DEV)
        chosen_ids, w, _ = R.route(view(leaf), None, top_k=4)
        got, = torch.autograd.grad(w, leaf, dw)
        want, = torch.autograd.grad(weights64(view(y), chosen_ids, 5.0, False, "sigmoid"), y, dw.double())
        assert bool(((got.double() - want).abs() <= TOL * 5 * dw.abs().double().sum()).all())


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("T,E", [(160001, 8), (320003, 16), (80001, 520), (155000, 1000)])
def test_balance_of_batches_beyond_32_tokens_per_warp(T, E, masked):
    """A warp fetches its masks for 32 tokens at a time: batches in which it has more of them, masked and not. An expert's sum
    of p (positive terms) goes through at most T / 2368 additions of a warp (148 CTAs of 16 warps or more), 32 over the
    warps, 5 over the parts of a thread and 5 of a tree, each off by 2^-24 of the sum at most: added to TOL. The
    gradient has no sum over tokens."""
    import router as R
    g = seeded(T + E)
    x = torch.randn(T, E, generator=g, device=DEV, requires_grad=True)
    ids = torch.randint(0, E, (T, 2), generator=g, device=DEV)
    mask = torch.rand(T, generator=g, device=DEV) < 0.7 if masked else None
    keep = mask if masked else torch.ones(T, dtype=torch.bool, device=DEV)
    for score in ("sigmoid", "softmax"):
        loss, n = R.balance_loss(x, ids, mask, score, 0.5)
        got, = torch.autograd.grad(loss, x)
        y = x.detach().double()
        want, n64, c = loss64(y, ids, mask, score, 0.5)
        assert torch.equal(n, n64.to(torch.int32))
        assert abs(float(loss.detach()) - float(want)) <= (TOL + (T / 2368 + 42) * 2.0 ** -24) * float(want)
        s = torch.sigmoid(y) if score == "sigmoid" else torch.softmax(y, -1)
        p = s / s.sum(-1, keepdim=True)
        dot = (c * p).sum(-1, keepdim=True)
        ref = p * (c - dot) * (1 - s if score == "sigmoid" else 1.0)
        error = (got.double() - ref).abs() - TOL * p * (c + dot)
        assert float(error[keep].max()) <= 0 and not got[~keep].any()
        assert bool(got[keep][-1].any())


def test_softmax_groups_left_out_are_never_chosen():
    """Kept groups with fewer finite logits than top_k: their experts at -inf, of the type's lowest value or NaN follow, by
    value and then by id; the left-out groups' experts do not, however large their softmax weight. The reference sorts
    (kept, value) pairs."""
    import router as R
    g = seeded(91)
    for E, n_group, kept, k in ((32, 4, 2, 12), (96, 8, 3, 32), (512, 8, 4, 22), (1024, 32, 2, 32), (160, 8, 1, 20)):
        size = E // n_group
        x = torch.randn(40, n_group, size, generator=g, device=DEV)
        strong = torch.argsort(torch.rand(40, n_group, generator=g, device=DEV), dim=1)[:, :kept]    # the groups to keep
        keep = torch.zeros(40, n_group, dtype=torch.bool, device=DEV).scatter_(1, strong, True)
        x[..., :2] += 30.0 * keep[..., None]
        x[..., 2:] = torch.where(keep[..., None] & (torch.rand(x[..., 2:].shape, generator=g, device=DEV) < 0.95), -float("inf"), x[..., 2:])
        x[5:10, :, size - 1] = torch.where(keep[5:10], torch.finfo(torch.float32).min, x[5:10, :, size - 1])
        x[10:15] = torch.where(keep[10:15, :, None] & (x[10:15] == -float("inf")) & (torch.arange(size, device=DEV) % 2 == 0), float("nan"), x[10:15])
        x[20, :, 1:] = -float("inf")                       # no group has a sum: the first ones are kept
        keep[20] = torch.arange(n_group, device=DEV) < kept
        flat, on = x.reshape(40, E), keep.repeat_interleave(size, 1)
        value = torch.where(torch.isnan(flat), -float("inf"), flat)
        by_value = torch.sort(value, dim=1, descending=True, stable=True)[1]
        first = torch.sort(on.gather(1, by_value).to(torch.int8), dim=1, descending=True, stable=True)[1]
        want = by_value.gather(1, first)[:, :k]
        leaf = flat.clone().requires_grad_()
        ids, w, n = R.route(leaf, None, top_k=k, n_group=n_group, topk_group=kept, score="softmax")
        assert bool(on.gather(1, ids).all()) and torch.equal(ids, want)
        assert torch.equal(n, torch.bincount(ids.flatten(), minlength=E).to(torch.int32))
        ref = weights64(flat.double(), ids, 5.0, False, "softmax")
        assert torch.allclose(w.detach().double(), ref, rtol=TOL, atol=5e-30, equal_nan=True)
        assert not w.detach()[:5][flat[:5].gather(1, ids[:5]) == -float("inf")].any()


def test_forward_mode_tangents_are_refused_without_grad_mode_too():
    import _qmoe_lib as C
    import router as R
    import torch.autograd.forward_ad as fwd
    x = torch.randn(6, 32, generator=seeded(92), device=DEV)
    ids = torch.topk(x, 3)[1]
    for grad in (True, False):
        with fwd.dual_level(), torch.set_grad_enabled(grad):
            dual = fwd.make_dual(x, torch.ones_like(x))
            for bad in (lambda: R.route(dual, None, top_k=3), lambda: R.balance_loss(dual, ids)):
                with pytest.raises(C.QmoeError, match="forward-mode"):
                    bad()
            assert not R.route(x, None, top_k=3)[1].requires_grad and not R.balance_loss(x, ids)[0].requires_grad


@pytest.mark.parametrize("k", [1, 22, 32])
@pytest.mark.parametrize("E", [96, 512])
def test_route_weights_of_ties_and_strange_numbers(E, k):
    """Saturated, tied, infinite, signed-zero and NaN rows: the weights are torch's own bits at the chosen experts (a NaN
    where torch has one), and a softmax's are those of 64 bits, NaN for rows that have none. Scores below fp32's normal
    numbers, 1.2e-38, may be 0: over the sum's 1e-20 and times 5 that is 6e-18 of a weight."""
    import router as R
    g = seeded(E)
    x = torch.randn(16, E, generator=g, device=DEV)
    x[0] = 0.0
    x[1, 40:] = 1.0
    x[2], x[3] = -200.0, 200.0
    x[4, ::2] = -float("inf")
    x[5, 10], x[5, 90] = float("inf"), -float("inf")
    x[6, 3:60] = float("nan")
    x[7] = torch.arange(E, device=DEV) % 3
    x[8], x[8, 50:] = -0.0, 0.0
    x[9] = float("nan")
    x[10] = -torch.arange(E, device=DEV).float()
    x[11] = 20.0 + torch.arange(E, device=DEV) % 96 * 0.1
    x[12, 5:] = -float("inf")
    x[13, 5:] = torch.finfo(torch.float32).min
    x[14] = -float("inf")
    for norm in (False, True):
        for bias in (None, torch.linspace(-1, 1, E, device=DEV)):
            ids, w, n = R.route(x, bias, top_k=k)
            assert torch.equal(ids, chosen(x, bias, k))
            assert torch.equal(torch.nan_to_num(w, nan=-1.0), torch.nan_to_num(torch.sigmoid(x).gather(1, ids) * 5.0, nan=-1.0))
            ids, w, _ = R.route(x, bias, top_k=k, norm_topk_prob=True)
            assert torch.allclose(w.double(), weights64(x.double(), ids, 5.0, True, "sigmoid"), rtol=TOL, atol=5e-17, equal_nan=True)
        ids, w, n = R.route(x, None, top_k=k, score="softmax", norm_topk_prob=norm)
        assert torch.equal(ids, chosen(x, None, k, score="softmax"))
        assert torch.allclose(w.double(), weights64(x.double(), ids, 5.0, norm, "softmax"), rtol=TOL, atol=5e-17 if norm else 5e-30, equal_nan=True)
