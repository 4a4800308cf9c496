"""Four-bit quantisation and product (dense_q.quantize / gemm / qlinear_a4) against their definition in 64 bits.

Quantisation is exact: codes, scales and s have to be the definition's, ties included. The product's terms are exact and
its sums run in fp32: with K terms, each addition off by at most one last place (2^-23 of the sum of magnitudes),
|y - exact| <= K 2^-23 sum |x w|, and half a step of the output type for the final rounding. With small integers every
partial sum is a 24-bit number and the result has to be equal."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
E2M1 = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)


def seeded(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def nearest_even(v, step):
    return torch.round(v / step) * step


def definition(x, per_row):
    """(values of the codes, scales, s) in 64 bits."""
    x = x.double()
    M, K = x.shape
    a = torch.where(torch.isfinite(x), x.abs(), 0.0)
    top = a.amax(1) if per_row else a.max().reshape(1)
    m, e = torch.frexp(top)
    e = torch.where(m * 2 <= 1.3125, e - 12, e - 11).clamp(min=-126)
    s = torch.ldexp(torch.ones_like(top), torch.where(top > 0, e, -126))
    b = x.reshape(M, K // 16, 16) / s[:, None, None]
    fine = torch.isfinite(b).all(-1)
    r = torch.where(torch.isfinite(b), b.abs(), 0.0).amax(-1) / 6
    step = torch.exp2(torch.frexp(r.clamp_min(2.0 ** -6))[1].double() - 4)
    sc = nearest_even(r, step)
    q = torch.where((sc > 0)[..., None], b / sc[..., None].clamp_min(1e-300), 0.0)
    q = torch.where(torch.isfinite(q), q, 0.0)
    step = torch.where(q.abs() < 2, 0.5, torch.where(q.abs() < 4, 1.0, 2.0)).double()
    v = nearest_even(q, step).clamp(-6, 6)
    return torch.where(fine[..., None], v, 0.0), torch.where(fine, sc, float("nan")), s


def codes_of(q):
    w = q["w"].long()
    return E2M1.to(DEV)[torch.stack([w & 15, w >> 4], -1)].reshape(q["N"], q["K"] // 16, 16)


def scales_of(q):
    return q["sc"].view(torch.float8_e4m3fn).double()


def values_of(q):
    s = q["s"].double().reshape(-1, 1, 1)
    return (codes_of(q) * scales_of(q)[..., None] * s).reshape(q["N"], q["K"])


def check_quantized(q, x, per_row):
    v, sc, s = definition(x, per_row)
    assert torch.equal(q["s"].double(), s)
    assert torch.equal(torch.nan_to_num(scales_of(q), nan=-1.0), torch.nan_to_num(sc, nan=-1.0))
    assert torch.equal(codes_of(q), v)
    if "sca" not in q:
        import dense_q as D
        q = D.prepare(q)
    # the same scales as atoms: row r of k-step ks at [r / 128][ks], (r % 32) * 16 + (r % 128 / 32) * 4
    M, nb = q["N"], q["K"] // 16
    nks = (nb + 3) // 4
    r = torch.arange(M, device=DEV)
    at = ((r // 128)[:, None] * nks + torch.arange(nks, device=DEV)) * 512 + ((r % 32) * 16 + (r % 128) // 32 * 4)[:, None]
    got = q["sca"][at[..., None] + torch.arange(4, device=DEV)].reshape(M, nks * 4)
    assert torch.equal(got[:, :nb], q["sc"]) and not got[:, nb:].any()


@pytest.mark.parametrize("per_row", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,K", [(1, 16), (1, 4096), (2, 48), (5, 32), (33, 2688), (129, 1024), (3, 2064), (7, 16400), (300, 208)])
def test_quantize(M, K, dtype, per_row):
    import dense_q as D
    g = seeded(M * K)
    x = torch.randn(M, K, generator=g, device=DEV) * torch.exp(2 * torch.randn(M, 1, generator=g, device=DEV))
    x = x.to(dtype)
    x[M // 2, K // 2:K // 2 + 16] = 0
    check_quantized(D.quantize(x, per_row, True), x, per_row)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantize_ties_and_borders(dtype):
    """Rows whose largest value sets s = 1 and each block's scale: exact ties of codes and of scales go to the even
    neighbour, and the next representable number on either side of a tie goes to its own side."""
    import dense_q as D
    rows = []
    for sc in (2.0 ** -9, 7 * 2.0 ** -9, 0.125, 0.140625, 1.0, 1.125, 1.25, 1.375, 1.5, 1.625, 1.75, 1.875, 15.0, 416.0, 448.0):
        mid = torch.tensor([6.0, .25, .75, 1.25, 1.75, 2.5, 3.5, 5.0, -.25, -.75, -1.25, -1.75, -2.5, -3.5, -5.0, 0.0]) * sc
        rows.append(mid)
        up = torch.nextafter(mid.to(dtype), torch.full_like(mid, float("inf")).to(dtype)).float()
        down = torch.nextafter(mid.to(dtype), torch.full_like(mid, -float("inf")).to(dtype)).float()
        up[0] = down[0] = 6.0 * sc
        rows += [up, down]
    sc = torch.arange(8, 127)
    table = torch.where(sc < 8, sc * 2.0 ** -9, (8 + sc % 8) * torch.exp2(sc.float() // 8 - 10))
    edge = (6 * (table[1:] + table[:-1]) / 2)          # ties between block scales
    for e in (edge, torch.nextafter(edge.to(dtype), torch.zeros_like(edge).to(dtype)).float(),
              torch.nextafter(edge.to(dtype), torch.full_like(edge, 1e4).to(dtype)).float()):
        rows += [torch.cat([v.reshape(1), torch.zeros(15)]) for v in e]
    x = torch.stack(rows).to(dtype).to(DEV)
    top = torch.zeros(len(rows), 16, dtype=dtype, device=DEV)
    top[:, 3] = 2688.0                                  # s = 1
    x = torch.cat([x, top], 1).contiguous()
    q = D.quantize(x)
    assert torch.equal(q["s"], torch.ones_like(q["s"]))
    check_quantized(q, x, True)


@pytest.mark.parametrize("per_row", [True, False])
def test_quantize_extremes(per_row):
    """Zero rows, subnormals, the largest numbers, signed zeros, infinities and NaN."""
    import dense_q as D
    x = torch.zeros(12, 64, device=DEV)
    x[1] = 1e-45
    x[2] = 2.0 ** -130
    x[3, ::3] = 3.4028234663852886e38
    x[4] = torch.randn(64, generator=seeded(1), device=DEV) * 2.0 ** -126
    x[5] = -0.0
    x[6] = torch.randn(64, generator=seeded(2), device=DEV)
    x[6, 17] = float("nan")
    x[7] = x[6]
    x[7, 3], x[7, 17], x[7, 40] = float("inf"), 1.0, -float("inf")
    x[8] = float("nan")
    x[9, 63] = float("inf")
    x[10] = torch.randn(64, generator=seeded(3), device=DEV) * 1e30
    x[11, 5] = -1e-30
    q = D.quantize(x, per_row)
    check_quantized(q, x, per_row)
    back = D.dequant(q).float()
    assert torch.isnan(back[6, 16:32]).all() and torch.isfinite(back[6, :16]).all() and torch.isfinite(back[6, 32:]).all()
    for dt in (torch.bfloat16, torch.float16):
        y = x[6:8].to(dt)
        check_quantized(D.quantize(y, per_row, True), y, per_row)


def test_quantize_strides_and_offsets():
    import dense_q as D
    base = torch.randn(70, 1100, generator=seeded(9), device=DEV).to(torch.bfloat16)
    for x in (base[:, :1024], base[::3, 1:993], base[:, 8:1032], base.t()[:64].t()[:, :64], base.view(-1)[16:16 + 65 * 1104].view(65, 1104)[:, :1088], base[:1, :1088], base.t()[:1088, :64].t()):
        check_quantized(D.quantize(x, for_gemm=True), x, True)
        check_quantized(D.quantize(x, per_row=False), x, False)
    one = base[0, :16].reshape(1, 16).expand(5, 16)      # a broadcast row
    check_quantized(D.quantize(one), one, True)
    empty = D.quantize(base[:0, :64])
    assert empty["w"].shape == (0, 32) and D.dequant(empty).shape == (0, 64)
    assert D.gemm(D.quantize(base[:4, :64]), empty).shape == (0, 4) and D.gemm(empty, D.quantize(base[:4, :64])).shape == (4, 0)


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("per_row", [True, False])
def test_dequantize(out, per_row):
    import dense_q as D
    x = torch.randn(37, 2688, generator=seeded(4), device=DEV)
    q = D.quantize(x, per_row)
    buf = torch.empty(37 * 2688 + 1, dtype=out, device=DEV)
    for at in (0, 1):                                   # aligned and not
        y = D.dequant_rows(q, 3, 30, buf[at:at + 27 * 2688].view(27, 2688))
        assert torch.equal(y, values_of(q)[3:30].float().to(out))
    assert torch.equal(D.dequant(q), values_of(q).float().to(torch.bfloat16))


# ------------------------------------------------------------------------------------------------ product
def small_integers(g, rows, K):
    """Random codes and scales 0.5, 1, 2: every product is a multiple of 1/16, every sum a 24-bit number."""
    w = torch.randint(0, 256, (rows, K // 2), generator=g, device=DEV, dtype=torch.uint8)
    sc = torch.tensor([0x30, 0x38, 0x40], dtype=torch.uint8, device=DEV)[torch.randint(0, 3, (rows, K // 16), generator=g, device=DEV)]
    return {"fmt": "nvfp4", "w": w, "sc": sc.contiguous(), "s": torch.ones(1, device=DEV), "N": rows, "K": K}


SHAPES = [(1, 128, 32), (1, 2688, 4096), (1, 1, 64), (2, 127, 96), (15, 129, 256), (16, 300, 2688), (17, 1024, 1024), (31, 4096, 544),
          (33, 77, 4096), (64, 1000, 160), (65, 513, 2688), (100, 4096, 320), (128, 2688, 512), (129, 640, 1024), (200, 20000, 64),
          (255, 257, 4096), (256, 12288, 288), (300, 2688, 2688), (513, 4096, 1056), (1000, 1111, 4096), (2047, 2688, 96), (4100, 1300, 512)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_gemm_small_integers(M, N, K):
    import dense_q as D
    g = seeded(M + N + K)
    xq, q = small_integers(g, M, K), small_integers(g, N, K)
    xq["fmt"], xq["s"] = "nvfp4_rows", torch.exp2(torch.randint(-3, 4, (M,), generator=g, device=DEV).float())
    ref = values_of(xq) @ values_of(q).t()
    y = D.gemm(q, xq, torch.float32)
    assert torch.equal(y.double(), ref)
    assert torch.equal(D.gemm(D.prepare(q), D.prepare(xq), torch.bfloat16), ref.float().to(torch.bfloat16))
    assert D.gemm_status() == 0


def bound(xq, q, y):
    """Of |y - exact|: K additions, one last place of the sum of magnitudes each, and the type's half step."""
    mag = values_of(xq).abs() @ values_of(q).abs().t()
    return xq["K"] * 2.0 ** -23 * mag + torch.finfo(y.dtype).eps / 2 * y.double().abs()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,N,K", [(1, 2688, 4096), (3, 4096, 2688), (37, 4096, 2688), (130, 999, 1024), (600, 2688, 4096)])
def test_linear_against_64_bits(M, N, K, dtype):
    import dense_q as D
    g = seeded(M * 7 + N)
    x = (torch.randn(M, K, generator=g, device=DEV) * torch.exp(torch.randn(M, 1, generator=g, device=DEV))).to(dtype)
    q = D.quantize(torch.randn(N, K, generator=g, device=DEV) * 0.02, per_row=False)
    q["s"] = q["s"] * 1.37                              # a checkpoint's scale is no power of two
    xq = D.quantize(x)
    v, sc, s = definition(x, True)
    assert torch.equal(values_of(xq), (v * sc[..., None]).reshape(M, K) * s[:, None])
    ref = values_of(xq) @ values_of(q).t()
    y = D.qlinear_a4(q, x)
    assert y.dtype == dtype and bool(((y.double() - ref).abs() <= bound(xq, q, y)).all())
    # the epilogues, from the rounded product
    base = y.float()
    assert torch.equal(D.qlinear_a4(q, x, act="relu2"), (torch.relu(base) ** 2).to(dtype))
    res = torch.randn(M, N, generator=g, device=DEV).to(dtype)
    assert torch.equal(D.qlinear_a4(q, x, residual=res), (base + res.float()).to(dtype))
    assert torch.equal(D.qlinear_a4(q, x), y)           # the same bits again


def test_linear_shapes_and_row_scales():
    import dense_q as D
    g = seeded(77)
    q = D.prepare(D.quantize(torch.randn(96, 64, generator=g, device=DEV), per_row=True))
    x = torch.randn(2, 3, 64, generator=g, device=DEV).to(torch.bfloat16)
    y = D.qlinear_a4(q, x)
    assert y.shape == (2, 3, 96)
    xq = D.quantize(x.view(6, 64))
    ref = values_of(xq) @ values_of(q).t()
    assert bool(((y.view(6, 96).double() - ref).abs() <= bound(xq, q, y.view(6, 96))).all())
    assert D.qlinear_a4(q, x[:0]).shape == (0, 3, 96)
    assert D.qlinear_a4(q, x[0, 0]).shape == (96,)


def test_rows_do_not_depend_on_their_batch():
    """Each row's codes and scales are its own; with small integers the product is exact, so a row is the same alone."""
    import dense_q as D
    g = seeded(5)
    xq, q = small_integers(g, 700, 1024), D.prepare(small_integers(g, 640, 1024))
    y = D.gemm(q, xq, torch.float32)
    for lo, hi in ((0, 1), (3, 20), (100, 228), (5, 350)):
        part = {**xq, "w": xq["w"][lo:hi].clone(), "sc": xq["sc"][lo:hi].clone(), "N": hi - lo}
        assert torch.equal(D.gemm(q, part, torch.float32), y[lo:hi])


def test_nan_blocks_reach_only_their_row_and_column():
    import dense_q as D
    g = seeded(6)
    x = torch.randn(200, 512, generator=g, device=DEV).to(torch.bfloat16)
    w = torch.randn(300, 512, generator=g, device=DEV)
    clean = D.gemm(D.quantize(w, False), D.quantize(x))
    xb, wb = x.clone(), w.clone()
    xb[150, 7], wb[131, 500] = float("inf"), float("nan")
    y = D.gemm(D.quantize(wb, False), D.quantize(xb))
    bad = torch.zeros(200, 300, dtype=torch.bool, device=DEV)
    bad[150], bad[:, 131] = True, True
    assert torch.isnan(y[bad]).all() and torch.isfinite(y[~bad]).all()
    assert torch.equal(y[~bad], clean[~bad]) or float(w.abs().max()) == float(w[131].abs().max())


@pytest.mark.parametrize("M", [1, 40, 300])
def test_graph_replay_and_side_stream(M):
    import dense_q as D
    g = seeded(M)
    q = D.prepare(D.quantize(torch.randn(512, 1024, generator=g, device=DEV), False))
    xs = [torch.randn(M, 1024, generator=g, device=DEV).to(torch.bfloat16) for _ in range(3)]
    want = [D.qlinear_a4(q, x) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [D.qlinear_a4(q, x) for x in xs]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    buf = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = D.qlinear_a4(q, buf)
    for x, y in zip(xs, want):
        buf.copy_(x)
        graph.replay()
        assert torch.equal(out, y)


def test_a_wait_that_runs_out_is_reported_and_the_next_call_is_right():
    import dense_q as D
    import qmoe_ns as Q
    g = seeded(8)
    for M in (4, 500):
        xq, q = D.prepare(small_integers(g, M, 4096)), D.prepare(small_integers(g, 1024, 4096))
        ref = D.gemm(q, xq, torch.float32)
        torch.cuda.synchronize()
        Q.set_wait_cycles(1)
        try:
            D.gemm(q, xq, torch.float32)
            assert D.gemm_status() == 4
        finally:
            Q.set_wait_cycles(0)
        assert D.gemm_status() == 0
        assert torch.equal(D.gemm(q, xq, torch.float32), ref) and D.gemm_status() == 0


@pytest.mark.parametrize("M", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("N,K", [(1, 32), (3, 64), (17, 992), (2688, 4096), (300, 2080), (129, 16384), (100, 16416)])
def test_linear_of_few_tokens(M, N, K):
    """The one-kernel form (up to four rows) and the sizes beside it: the quantiser's own codes, strided rows, per-row
    weight scales, a NaN block and a row of zeros."""
    import dense_q as D
    g = seeded(M * K + N)
    q = D.prepare(D.quantize(torch.randn(N, K, generator=g, device=DEV) * 0.05, per_row=M % 2 == 0))
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        base = torch.randn(M, K + 8, generator=g, device=DEV).to(dtype)
        for x in (base[:, :K], base[:, 3:3 + K]):
            xq = D.quantize(x)
            ref = values_of(xq) @ values_of(q).t()
            y = D.qlinear_a4(q, x)
            assert bool(((y.double() - ref).abs() <= bound(xq, q, y)).all())
            assert torch.equal(D.qlinear_a4(q, x, act="relu2"), (torch.relu(y.float()) ** 2).to(dtype))
        x = base[:, :K].clone()
        x[M - 1] = 0
        x[0, 5] = float("nan")
        y = D.qlinear_a4(q, x)
        assert torch.isnan(y[0]).all() and torch.isfinite(y[1:]).all() and (M == 1 or not y[M - 1].any())


def test_residual_of_another_shape_is_refused():
    import _qmoe_lib as C
    import dense_q as D
    q = D.prepare(D.quantize(torch.ones(6, 64, device=DEV), False))
    x = torch.ones(2, 3, 64, device=DEV)
    D.qlinear_a4(q, x, residual=torch.ones(2, 3, 6, device=DEV))
    for shape in ((6, 6), (3, 2, 6), (1, 1, 6), (2, 3, 5)):
        with pytest.raises(C.QmoeError, match="residual"):
            D.qlinear_a4(q, x, residual=torch.ones(shape, device=DEV))
    with pytest.raises(C.QmoeError, match="residual"):
        D.qlinear_a4(q, x, residual=torch.ones(2, 3, 6, device=DEV, dtype=torch.float16))
    rows = {**q, "N": 5}
    with pytest.raises(C.QmoeError, match="w must"):
        D.qlinear_a4(rows, x)


def test_no_memory_is_torchs_own_error():
    import dense_q as D
    x = torch.zeros(1, 4096, device=DEV).expand(1 << 28, 4096)    # a copy would take 4 TB
    with pytest.raises(torch.OutOfMemoryError):
        D.quantize(x)
    assert torch.equal(D.quantize(x[:3])["s"], torch.full((3,), 2.0 ** -126, device=DEV))


def test_two_streams_at_once():
    """Calls of every form in flight on two streams: the same bits as one after the other."""
    import dense_q as D
    g = seeded(91)
    q = D.prepare(D.quantize(torch.randn(1000, 2048, generator=g, device=DEV), False))
    xs = [torch.randn(M, 2048, generator=g, device=DEV).to(torch.bfloat16) for M in (1, 3, 30, 60, 300, 700)]
    want = [D.qlinear_a4(q, x) for x in xs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got += [(j, D.qlinear_a4(q, xs[j])) for j in (range(len(xs)) if i else reversed(range(len(xs))))]
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[j]) for j, y in got) and D.gemm_status() == 0


@pytest.mark.parametrize("M,N,K", [(2048, 2688, 512), (512, 10000, 96), (300, 11000, 288), (600, 9001, 320), (577, 9001, 32)])
def test_gemm_in_one_wave_of_wide_tiles(M, N, K):
    """Sizes whose tiles of 256 x 320 are one per pair of SMs: tiles that start inside an atom, end in their first part or
    a few columns later, rows of y that are not aligned; the three types and epilogues, exact."""
    import dense_q as D
    g = seeded(M + N + K)
    xq, q = D.prepare(small_integers(g, M, K)), D.prepare(small_integers(g, N, K))
    ref = (values_of(xq) @ values_of(q).t()).float()
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        base = ref.to(dtype)
        res = torch.randint(-8, 8, (M, N), generator=g, device=DEV).to(dtype)
        assert torch.equal(D.gemm(q, xq, dtype), base)
        assert torch.equal(D.gemm(q, xq, dtype, act="relu2"), (torch.relu(base.float()) ** 2).to(dtype))
        assert torch.equal(D.gemm(q, xq, dtype, residual=res), (base.float() + res.float()).to(dtype))
    assert D.gemm_status() == 0


def test_the_inverse_refuses_what_it_cannot_read():
    """Scales that stayed on the CPU, outputs of another size; scales in their own type are the same bytes."""
    import _qmoe_lib as C
    import dense_q as D
    x = torch.randn(5, 64, generator=seeded(14), device=DEV)
    for per_row in (True, False):
        q = D.quantize(x, per_row)
        for name in ("w", "sc", "s"):
            with pytest.raises(C.QmoeError, match="one device"):
                D.dequant({**q, name: q[name].cpu()})
        assert torch.equal(D.dequant({**q, "sc": q["sc"].view(torch.float8_e4m3fn)}), D.dequant(q))
    q = D.quantize(x)
    for name in ("w", "sc", "s"):
        with pytest.raises(C.QmoeError, match="one device"):
            D.dequant_rows({**q, name: q[name].cpu()}, 0, 5, torch.empty(5, 64, device=DEV))
    for lo, hi, out in ((0, 5, torch.empty(4, 64, device=DEV)), (0, 5, torch.empty(5, 64)), (3, 2, torch.empty(1, 64, device=DEV)),
                        (3, 6, torch.empty(3, 64, device=DEV)), (-1, 2, torch.empty(3, 64, device=DEV))):
        with pytest.raises(C.QmoeError):
            D.dequant_rows(q, lo, hi, out)
    assert torch.equal(D.dequant_rows(q, 2, 4, torch.empty(2, 64, device=DEV)), values_of(q)[2:4].float())
    assert D.dequant_rows(q, 2, 2, torch.empty(0, 64, device=DEV)).numel() == 0


@pytest.mark.parametrize("M,N,K", [(100, 4096, 4096), (2000, 4096, 4096), (2048, 2688, 4096), (700, 4097, 2688), (700, 4097, 32768), (2048, 8192, 32768)])
def test_waits_that_run_out_anywhere_in_a_pair(M, N, K):
    """Limits from less than one copy's latency to more than the whole product: the two CTAs of a pair give up at stages of
    their own. Each call either reports it or is right, ends at once (the drain waits for what was issued, not for its
    2 s bound), and the next one is right. (A single poll of a barrier may outlast a short product: only the long ones
    surely give up.)"""
    import time

    import dense_q as D
    import qmoe_ns as Q
    g = seeded(M)
    xq, q = D.prepare(small_integers(g, M, K)), D.prepare(small_integers(g, N, K))
    ref = D.gemm(q, xq, torch.float32)
    assert D.gemm_status() == 0
    late = 0
    for limit in [1, 1, 100, 300, 600] + list(range(800, 6000, 200)) + list(range(6000, 30000, 2000)):
        Q.set_wait_cycles(limit)
        try:
            torch.cuda.synchronize()
            start = time.perf_counter()
            y = D.gemm(q, xq, torch.float32)
            status = D.gemm_status()
            assert time.perf_counter() - start < 1.0
        finally:
            Q.set_wait_cycles(0)
        late += status == 4
        assert status == 4 or (status == 0 and torch.equal(y, ref))
        assert torch.equal(D.gemm(q, xq, torch.float32), ref) and D.gemm_status() == 0
    assert late > 0 or K < 32768


@pytest.mark.parametrize("M", [1, 4, 5])
def test_linear_of_a_weight_that_was_not_prepared(M):
    """The same bits as with its scales laid out; few rows take one kernel and lay out nothing."""
    import dense_q as D
    g = seeded(M)
    q = D.quantize(torch.randn(300, 512, generator=g, device=DEV), False)
    x = torch.randn(M, 512, generator=g, device=DEV).to(torch.bfloat16)
    want = D.qlinear_a4(D.prepare(q), x)
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    y = D.qlinear_a4(q, x)
    assert torch.cuda.memory_stats()["allocation.all.allocated"] - before == (1 if M < 5 else 3)   # y; scales, workspace
    assert torch.equal(y, want)


def test_a_weight_that_changed_is_prepared_anew():
    """prepare lays out the scales that the dict holds now, an older "sca" or not: few and many rows then agree."""
    import dense_q as D
    g = seeded(15)
    q = D.prepare(small_integers(g, 200, 512))
    x = torch.randint(-2, 3, (5, 512), generator=g, device=DEV).float()
    part = {**q, "w": q["w"][40:100].clone(), "sc": q["sc"][40:100].clone(), "N": 60}
    q["sc"][:, 3] = 0x40
    for w in (D.prepare(part), D.prepare(q)):
        fresh = {k: v for k, v in w.items() if k != "sca"}
        xq = D.quantize(x)
        want = (values_of(xq) @ values_of(w).t()).float()
        assert torch.equal(D.qlinear_a4(w, x), want) and torch.equal(D.qlinear_a4(fresh, x), want)
        assert torch.equal(D.qlinear_a4(w, x[:4]), want[:4]) and torch.equal(D.gemm(w, xq, torch.float32), want)
