"""The MoE layer over a prompt (decode_step.MoELayer): with prompt_a4 the router, the quantiser, the four-bit products and
the routed experts together, as a user runs them; without it, what the layer gave before."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
H, LAT, SI, NE = 2048, 1024, 1344, 512


@pytest.fixture(scope="module")
def parts():
    import dense_q as D
    import expert_store as ES
    import qmoe_ns as Q
    import qmoe_synth as S
    g = S.seeded(77, DEV)
    blocks = torch.empty(NE, Q.BLOCK, dtype=torch.uint8, device=DEV)
    s2 = torch.empty(1, NE, 2, device=DEV)
    m_hat = S.unit_dir(g, DEV)
    for e0 in range(0, NE, 64):
        blk, s2b, _ = S.expert_blocks(64, 0.075, m_hat, g, DEV)
        blocks[e0:e0 + 64].copy_(blk)
        s2[0, e0:e0 + 64] = s2b
    Q.to_T_batch(blocks)
    store = ES.ExpertStore.from_tensors(blocks, s2, "T")

    def nvfp4(n, k):
        return D.quantize(torch.randn(n, k, generator=g, device=DEV) * 0.02, per_row=False)

    gate = (torch.randn(NE, H, generator=g, device=DEV) * 0.02).to(torch.bfloat16)
    bias = torch.randn(NE, generator=g, device=DEV) * 0.01
    codes, s = S.quantize_fp8(torch.randn(LAT, H, generator=g, device=DEV) * 0.02)
    fp8 = {"fmt": "fp8", "w": codes, "s": s.float(), "N": LAT, "K": H}
    return dict(store=store, gate=gate, bias=bias, fc1=nvfp4(LAT, H), fc2=nvfp4(H, LAT), up=nvfp4(SI, H), down=nvfp4(H, SI),
                fp8=fp8, g=g)


def layer_of(p, fc1="fc1", **kw):
    import decode_step as DS
    return DS.MoELayer(0, p["store"], p["gate"], p["bias"], p[fc1], p["fc2"], p["up"], p["down"], **kw)


@pytest.mark.parametrize("T", [5, 64, 301])
@pytest.mark.parametrize("fc1", ["fc1", "fp8"])
def test_four_bit_prompt(parts, T, fc1):
    """Bit for bit the parts called one by one; the experts and their counts those of the torch router."""
    import decode_step as DS
    import dense_q as D
    layer = layer_of(parts, fc1, prompt_a4=True)
    x = torch.randn(1, T, H, generator=parts["g"], device=DEV).to(torch.bfloat16)
    out = layer(x)
    x2 = x[0]
    ids_t, w_t = DS.route_tokens(x2, layer.gate_w, layer.bias)
    assert torch.equal(layer.counts, torch.bincount(ids_t.flatten(), minlength=NE).to(torch.int32))
    order = torch.argsort(torch.sigmoid(torch.nn.functional.linear(x2.float(), layer.gate_w)).gather(1, ids_t) +
                          layer.bias[ids_t], dim=1, descending=True, stable=True)
    ids, w = ids_t.gather(1, order), w_t.gather(1, order)
    lat = D.qlinear_a4(parts["fc1"], x2) if fc1 == "fc1" else D.qlinear(parts["fp8"], x2)
    y = layer.experts(lat, ids, w)
    base = D.gemm(parts["fc2"], D.quantize(y))
    u = torch.relu(D.gemm(parts["up"], D.quantize(x2)))
    want = base + D.gemm(parts["down"], D.quantize(u * u))
    assert out.shape == x.shape and torch.equal(out[0], want)
    assert torch.equal(layer(x), out)
    # Only the activations' rounding stands between it and the layer without it: at most a step of e2m1 / 4 of a value,
    # about 0.1 of a row in each product, twice that through a squared ReLU; four of them on the longer way, under 0.35.
    ref = layer_of(parts, fc1)(x)
    assert float((out.float() - ref.float()).norm() / ref.float().norm()) < 0.35


def test_prompt_without_the_flag_is_what_it_was(parts):
    import decode_step as DS
    import dense_q as D
    layer = layer_of(parts)
    x = torch.randn(40, H, generator=parts["g"], device=DEV).to(torch.bfloat16)
    ids, w = DS.route_tokens(x, layer.gate_w, layer.bias)
    lat = D.qlinear(parts["fc1"], x)
    out = D.qlinear(parts["fc2"], layer.experts(lat, ids, w))
    u = torch.relu(D.qlinear(parts["up"], x))
    assert torch.equal(layer(x), out + D.qlinear(parts["down"], u * u)) and layer.counts is None


def test_few_tokens_keep_their_path(parts):
    x = torch.randn(4, H, generator=parts["g"], device=DEV).to(torch.bfloat16)
    a, b = layer_of(parts), layer_of(parts, prompt_a4=True)
    for t in (1, 2, 4):
        assert torch.equal(a(x[:t]), b(x[:t]))


def test_prompt_as_a_graph(parts):
    layer = layer_of(parts, prompt_a4=True)
    xs = [torch.randn(96, H, generator=parts["g"], device=DEV).to(torch.bfloat16) for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(xs[0])
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    want = [layer(x).clone() for x in xs]
    buf = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = layer(buf)
    for x, y in zip(xs, want):
        buf.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, y)
