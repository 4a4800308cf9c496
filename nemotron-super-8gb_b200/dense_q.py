"""Drop-in replacement of the reference's `dense_q` module (helgard-orlm/nemotron-super-8gb dense_q.py):
the dense part of Nemotron kept in its checkpoint formats (FP8 e4m3 per-tensor scale; NVFP4 = e2m1 +
e4m3 per 16 + weight_scale_2), multiplied by libqmoe_b200's sm_100a GEMV kernels.

Same quantized-weight dict {"fmt", "w", "sc", "s", "N", "K"} (dense_q.py:237-247), same functions.
Dispatch (dense_q.py:215-234): M == 1 -> gemv; 2 <= M <= MB_MAX -> gemv_mb (weights read once for all
vectors; the reference's limit is 2, these kernels take up to 4); larger M -> exact dequantization to
bf16 in row chunks (dq_dequant_rows) + F.linear (cuBLAS), as the reference does.

Four-bit activations: `quantize` makes the same dict from a tensor, with one scale ("nvfp4", a weight) or one per row
("nvfp4_rows", activations: a row's result does not depend on the other rows); `gemm` multiplies two of them on the
tensor cores, and `qlinear_a4` is both, a linear that quantizes its input. `prepare` lays a loaded weight's scales
out for `gemm` once. These are inference operators: they refuse inputs that need a gradient.
"""
import types

import torch
import torch.nn.functional as F

import _qmoe_lib as C

SCR_MIB = 64
_SCR = {}
MB_ON = True
MB_MAX = 4
# Kept for API compatibility (dense_q.py:156-164); the CUDA kernels choose their own launch shapes.
CFG = {"fp8": dict(BLOCK_N=16, BK=256, NSPLIT=1, num_warps=4), "nvfp4": dict(BLOCK_N=16, GB=8, NSPLIT=1, num_warps=2)}
CFG_BY_SHAPE = {}
E2M1_T = None


def _gemv(q, x2, M):
    N, K = q["N"], q["K"]
    if q["fmt"] == "nvfp4_rows":
        raise C.QmoeError("the GEMVs take one scale per weight; this one has a scale per row (use gemm)")
    x2 = x2.contiguous()
    out = torch.empty(M, N, dtype=torch.float32, device=x2.device)
    st = C.stream_of(x2)
    if q["fmt"] == "fp8":
        C.call("dq_gemv_fp8", C.ptr(q["w"]), C.ptr(q["s"]), C.ptr(x2), C.dtype_code(x2), M, N, K, C.ptr(out), st)
    else:
        C.call("dq_gemv_nvfp4", C.ptr(q["w"]), C.ptr(q["sc"]), C.ptr(q["s"]), C.ptr(x2), C.dtype_code(x2), M, N, K,
               C.ptr(out), st)
    return out


def gemv(q, x):
    """dense_q.py:199-212: x [K] (any float) -> y float32 [N]."""
    return _gemv(q, x.reshape(1, -1), 1)[0]


def gemv_mb(q, x):
    """dense_q.py:139-152: x [M,K], M <= MB_MAX -> y float32 [M,N]; the weight is read once."""
    M = x.shape[0]
    assert M <= MB_MAX
    return _gemv(q, x, M)


def _lut(dev):
    """dense_q.py:170-176 (kept for callers that use the table directly)."""
    global E2M1_T
    if E2M1_T is None or E2M1_T.device != torch.device(dev):
        v = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float32,
                         device=dev)
        a = torch.arange(256, device=dev)
        E2M1_T = torch.stack([v[a & 15], v[a >> 4]], -1)
    return E2M1_T


def dequant_rows(q, r0, r1, out):
    """dense_q.py:179-188: rows [r0, r1) -> out [r1-r0, K] (bf16, fp16 or fp32), bit-exact."""
    if not out.is_contiguous():
        raise C.QmoeError("out must be contiguous")
    sc = q.get("sc")
    if q["fmt"] == "nvfp4_rows":
        if r1 > r0:
            with _on(out):
                C.call("dq_dequant_nvfp4", C.ptr(q["w"]), C.ptr(sc), C.ptr(q["s"]), 1, q["N"], q["K"], r0, r1, C.ptr(out),
                       C.dtype_code(out), C.stream_of(out))
        return out
    C.call("dq_dequant_rows", 0 if q["fmt"] == "fp8" else 1, C.ptr(q["w"]), C.ptr(sc) if sc is not None else None,
           C.ptr(q["s"]), q["N"], q["K"], r0, r1, C.ptr(out), C.dtype_code(out), C.stream_of(out))
    return out


def dequant(q):
    """dense_q.py:191-196: whole weight -> bf16 [N, K]."""
    out = torch.empty(q["N"], q["K"], dtype=torch.bfloat16, device=q["w"].device)
    return dequant_rows(q, 0, q["N"], out)


def qlinear(q, x):
    """dense_q.py:215-234: like F.linear(x, W_bf16) without bias: [..., K] -> [..., N] in x.dtype."""
    sh = x.shape
    x2 = x.reshape(-1, sh[-1])
    M, N = x2.shape[0], q["N"]
    if M == 1:
        return gemv(q, x2[0]).to(x.dtype).view(*sh[:-1], N)
    if M <= MB_MAX and MB_ON:
        return gemv_mb(q, x2).to(x.dtype).view(*sh[:-1], N)
    dev = x.device
    rows = max(1, min(N, SCR_MIB * 2**20 // (2 * q["K"])))
    scr = _SCR.get(dev)
    if scr is None or scr.numel() < rows * q["K"]:
        scr = _SCR[dev] = torch.empty(SCR_MIB * 2**20 // 2, dtype=torch.bfloat16, device=dev)
    y = torch.empty(M, N, dtype=x.dtype, device=dev)
    for r in range(0, N, rows):
        r1 = min(r + rows, N)
        w = dequant_rows(q, r, r1, scr[:(r1 - r) * q["K"]].view(r1 - r, q["K"]))
        y[:, r:r1] = F.linear(x2, w.to(x.dtype) if x.dtype != torch.bfloat16 else w)
    return y.view(*sh[:-1], N)


def load_q(ck, base, dev):
    """dense_q.py:237-247: checkpoint tensors under `base` -> quantized dict on `dev`, or None."""
    w = ck.get(base + ".weight")
    if base + ".weight_scale_2" in ck:
        sc = ck.get(base + ".weight_scale")
        return {"fmt": "nvfp4", "w": w.to(dev), "sc": sc.view(torch.uint8).to(dev),
                "s": ck.get(base + ".weight_scale_2").float().reshape(1).to(dev), "N": w.shape[0], "K": w.shape[1] * 2}
    if base + ".weight_scale" in ck and w.dtype == torch.float8_e4m3fn:
        return {"fmt": "fp8", "w": w.view(torch.uint8).to(dev),
                "s": ck.get(base + ".weight_scale").float().reshape(1).to(dev), "N": w.shape[0], "K": w.shape[1]}
    return None


def _fwd(self, x):
    return qlinear(self._q, x)


def attach(lin, q):
    """dense_q.py:254-261: nn.Linear -> quantized: the bf16 weight is released, forward goes to qlinear,
    .weight becomes the quantized bytes on the device."""
    assert lin.bias is None
    lin._parameters.pop("weight", None)
    lin._q = q
    object.__setattr__(lin, "weight", q["w"])
    lin.forward = types.MethodType(_fwd, lin)


class _on:
    """The tensor's device as the current one, for the launch (nothing to do where it is)."""
    __slots__ = ("dev", "was")

    def __init__(self, t):
        self.dev = t.get_device()

    def __enter__(self):
        self.was = torch._C._cuda_getDevice()
        if self.was != self.dev:
            torch.cuda.set_device(self.dev)

    def __exit__(self, *a):
        if self.was != self.dev:
            torch.cuda.set_device(self.was)


def _atoms_bytes(rows, K):
    return (rows + 127) // 128 * ((K + 63) // 64) * 512


def _no_grad(t):
    if t.requires_grad and torch.is_grad_enabled():
        raise C.QmoeError("the four-bit operators have no gradient: call them under torch.no_grad()")


def _rows(x):
    """A matrix as the kernels read it: unit column stride, rows that do not overlap; its dtype code and row stride."""
    _no_grad(x)
    C.ptr(x)
    dt = C.dtype_code(x)
    M, K = x.shape
    if x.is_contiguous():
        return x, dt, K
    if x.stride(1) != 1 or (M > 1 and x.stride(0) < K):
        x = x.contiguous()
    return x, dt, x.stride(0) if M > 1 else K


def quantize(x, per_row=True, for_gemm=False):
    """x [M, K] (bf16, fp16 or fp32; K a multiple of 16; rows may be strided) -> quantized dict: codes "w" [M, K/2],
    block scales "sc" [M, K/16] (e4m3 bytes), "s" f32 [M] with fmt "nvfp4_rows" (per_row), or [1] with fmt "nvfp4"
    (one scale for the tensor: a weight of this module); with for_gemm also "sca", the scales as gemm reads them (what
    prepare adds, in the same pass). s is the smallest power of two with amax <= 2688 s, scales and codes the nearest, ties to even. A 16-element block that holds an
    infinity or a NaN reads back as NaN; the others are as if that value were zero."""
    if x.dim() != 2:
        raise C.QmoeError("quantize takes a matrix [M, K]")
    M, K = x.shape
    if K < 16 or K % 16:
        raise C.QmoeError(f"quantize takes rows of a positive multiple of 16 elements (got {K})")
    if M == 0 and not per_row:
        raise C.QmoeError("a tensor without rows has no scale")
    x, dt, ld = _rows(x)
    dev = x.device
    w = torch.empty(M, K // 2, dtype=torch.uint8, device=dev)
    sc = torch.empty(M, K // 16, dtype=torch.uint8, device=dev)
    s = torch.empty(M if per_row else 1, dtype=torch.float32, device=dev)
    q = {"fmt": "nvfp4_rows" if per_row else "nvfp4", "w": w, "sc": sc, "s": s, "N": M, "K": K}
    sca = None
    if for_gemm:
        q["sca"] = torch.empty(_atoms_bytes(M, K), dtype=torch.uint8, device=dev)
        sca = q["sca"].data_ptr()
    if M:
        with _on(x):
            C.call("dq_quantize_nvfp4", x.data_ptr(), dt, ld, M, K, int(per_row), w.data_ptr(), sc.data_ptr(), s.data_ptr(), sca,
                   C.stream_of(x))
    return q


_NVFP4 = ("nvfp4", "nvfp4_rows")


def prepare(q):
    """A weight ready for gemm: the dict with "sca", its block scales as the tensor cores read them, added (the
    other tensors are shared with q)."""
    if q["fmt"] not in _NVFP4:
        raise C.QmoeError(f"gemm takes NVFP4 weights (got {q['fmt']})")
    if "sca" in q:
        return q
    N, K = q["N"], q["K"]
    for k, shape in (("w", (N, K // 2)), ("sc", (N, K // 16))):
        if q[k].dtype != torch.uint8 or q[k].shape != shape or not q[k].is_contiguous():
            raise C.QmoeError(f"{k} must be contiguous uint8 {list(shape)}")
    if q["s"].dtype != torch.float32 or q["s"].numel() != (N if q["fmt"] == "nvfp4_rows" else 1) or not q["s"].is_contiguous():
        raise C.QmoeError("s must be float32, one value (nvfp4) or one per row (nvfp4_rows)")
    if N == 0:
        return {**q, "sca": torch.empty(0, dtype=torch.uint8, device=q["sc"].device)}
    sc = q["sc"]
    C.ptr(sc)
    sca = torch.empty(_atoms_bytes(N, K), dtype=torch.uint8, device=sc.device)
    with _on(sc):
        C.call("dq_scale_atoms", C.ptr(sc), N, K, C.ptr(sca), C.stream_of(sc))
    return {**q, "sca": sca}


_ACTS = {None: 0, "relu2": 1}


def _check_product(q, M, K, dtype, dev, act, residual):
    """The epilogue's code, and the residual as the kernels read it."""
    if q["fmt"] not in _NVFP4:
        raise C.QmoeError(f"gemm takes NVFP4 operands (got {q['fmt']})")
    if q["K"] != K:
        raise C.QmoeError(f"gemm: {K} elements per activation row, {q['K']} per weight row")
    if K % 32 or K == 0:
        raise C.QmoeError(f"gemm takes rows of a positive multiple of 32 elements (got {K})")
    if act not in _ACTS or (act is not None and residual is not None):
        raise C.QmoeError("gemm: act is None or 'relu2', and not together with a residual")
    if dtype not in C.DT:
        raise C.QmoeError(f"unsupported output dtype {dtype}")
    if q["w"].device != dev:
        raise C.QmoeError(f"gemm: weight on {q['w'].device}, activations on {dev}")
    if residual is None:
        return _ACTS[act], None
    _no_grad(residual)
    if residual.shape != (M, q["N"]) or residual.dtype != dtype or residual.device != dev:
        raise C.QmoeError("gemm: the residual is [M, N] in the output's dtype, on its device")
    return 2, residual.contiguous()


def gemm(q, xq, dtype=torch.bfloat16, act=None, residual=None):
    """y [M, N] in dtype = dequant(xq) @ dequant(q).T for two NVFP4 dicts (xq of quantize: activations; q: a weight,
    either without "sca" has its scales laid out in this call), products exact, fp32 sums in a
    fixed order. act "relu2": relu(y)^2; residual [M, N] in dtype: y + residual; each on y rounded to dtype, as the
    unfused torch operators. K a multiple of 32."""
    if xq["fmt"] not in _NVFP4:
        raise C.QmoeError(f"gemm takes NVFP4 operands (got {xq['fmt']})")
    M, N, K = xq["N"], q["N"], xq["K"]
    dev = xq["w"].device
    ep, residual = _check_product(q, M, K, dtype, dev, act, residual)
    y = torch.empty(M, N, dtype=dtype, device=dev)
    if M == 0 or N == 0:
        return y
    q, xq = prepare(q), prepare(xq)
    with _on(y):
        C.call("dq_gemm_nvfp4", C.ptr(q["w"]), C.ptr(q["sca"]), C.ptr(q["s"]), int(q["fmt"] == "nvfp4_rows"),
               C.ptr(xq["w"]), C.ptr(xq["sca"]), C.ptr(xq["s"]), int(xq["fmt"] == "nvfp4_rows"), M, N, K, ep,
               C.ptr(residual), C.ptr(y), C.DT[dtype], C.stream_of(y))
    return y


def qlinear_a4(q, x, act=None, residual=None):
    """qlinear with the activations in NVFP4 too: x [..., K] is quantized row by row, then multiplied as gemm does:
    [..., N] in x.dtype (residual of that shape). The result carries the activations' four-bit rounding (about a tenth
    of a row's norm) and takes a fraction of a bf16 product's time."""
    sh = x.shape
    K, N = sh[-1], q["N"]
    x, dt, ld = _rows(x if len(sh) == 2 else x.reshape(-1, K))
    M, dev = x.shape[0], x.device
    if residual is not None:
        residual = residual.reshape(-1, N)
    ep, residual = _check_product(q, M, K, x.dtype, dev, act, residual)
    y = torch.empty(M, N, dtype=x.dtype, device=dev)
    if M and N:
        q = prepare(q)
        n, ws = 0, None
        if M > 4 or K > 16384:
            n = M * (K // 2) + _atoms_bytes(M, K) + (M + 3) // 4 * 16 + M * (K // 16)   # dq_linear_a4_workspace_bytes
            ws = torch.empty(n, dtype=torch.uint8, device=dev)
        with _on(x):
            C.call("dq_linear_a4", q["w"].data_ptr(), q["sc"].data_ptr(), q["sca"].data_ptr(), q["s"].data_ptr(), int(q["fmt"] == "nvfp4_rows"),
                   x.data_ptr(), dt, ld, M, N, K, ep, residual.data_ptr() if residual is not None else None, y.data_ptr(),
                   ws.data_ptr() if ws is not None else None, n, C.stream_of(x))
    return y if len(sh) == 2 else y.view(*sh[:-1], N)


def gemm_status(device=None, clear=True):
    """0, or the first error the gemm kernels of the device recorded since the last clear (a wait that ran out: 4, see
    qmoe_ns.set_wait_cycles); waits for the current stream."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    with torch.cuda.device(dev):
        return int(C.lib().dq_gemm_nvfp4_status(int(clear), torch.cuda.current_stream(dev).cuda_stream))


def nbytes(q):
    return sum(t.numel() * t.element_size() for k, t in q.items() if isinstance(t, torch.Tensor))
