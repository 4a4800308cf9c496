"""What the four-bit operators refuse, checked without a GPU: the C entry points' codes and the Python errors."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    import os

    import _qmoe_lib
    if not os.path.exists(_qmoe_lib.LIB_PATH):
        import qmoe_build
        qmoe_build.build()
    return _qmoe_lib.lib()


P = ctypes.c_void_p


def test_quantize_arguments(lib):
    a = P(256)

    def call(x=a, dt=1, ldx=64, M=4, K=64, w=a, sc=a, s=a, atoms=a):
        return lib.dq_quantize_nvfp4(x, dt, ldx, M, K, 1, w, sc, s, atoms, None)

    assert call(x=None) == 5 and call(w=None) == 5 and call(sc=None) == 5 and call(s=None) == 5
    assert call(M=0) == 1 and call(K=0) == 1 and call(K=40) == 1 and call(ldx=63) == 1 and call(M=1 << 31) == 1
    assert call(dt=3) == 6 and call(dt=9) == 6
    assert call(x=P(257)) == 2 and call(w=P(260)) == 2 and call(atoms=P(258)) == 2 and call(dt=0, x=P(258)) == 2
    if not torch.cuda.is_available():
        assert call() == 7 and call(atoms=None) == 7


def test_atoms_and_dequant_arguments(lib):
    a = P(256)
    assert lib.dq_scale_atoms(None, 4, 64, a, None) == 5
    assert lib.dq_scale_atoms(a, 0, 64, a, None) == 1 and lib.dq_scale_atoms(a, 4, 65, a, None) == 1
    assert lib.dq_scale_atoms(a, 4, 64, P(258), None) == 2
    assert lib.dq_dequant_nvfp4(a, a, a, 1, 4, 64, 3, 2, a, 1, None) == 1
    assert lib.dq_dequant_nvfp4(a, a, a, 1, 4, 64, 0, 5, a, 1, None) == 1
    assert lib.dq_dequant_nvfp4(P(257), a, a, 1, 4, 64, 0, 4, a, 1, None) == 2
    assert lib.dq_dequant_nvfp4(a, a, a, 1, 4, 64, 0, 4, a, 7, None) == 6


def test_gemm_arguments(lib):
    a = P(256)

    def call(w=a, wa=a, x=a, xa=a, M=4, N=8, K=64, ep=0, res=None, y=a, dt=1):
        return lib.dq_gemm_nvfp4(w, wa, a, 0, x, xa, a, 1, M, N, K, ep, res, y, dt, None)

    assert call(w=None) == 5 and call(xa=None) == 5 and call(y=None) == 5 and call(ep=2) == 5
    assert call(M=0) == 1 and call(N=0) == 1 and call(K=16) == 1 and call(K=48) == 1 and call(ep=3) == 1
    assert call(dt=3) == 6
    assert call(w=P(264)) == 2 and call(xa=P(264)) == 2 and call(y=P(257)) == 2 and call(dt=0, y=P(258)) == 2
    if not torch.cuda.is_available():
        assert call() == 7


def test_python_refusals():
    import _qmoe_lib as C
    import dense_q as D
    x = torch.zeros(2, 64)
    for bad in (torch.zeros(64), torch.zeros(2, 40), torch.zeros(2, 0), x, torch.zeros(2, 64, dtype=torch.float64)):
        with pytest.raises(C.QmoeError):
            D.quantize(bad)
    with pytest.raises(C.QmoeError):
        D.quantize(torch.zeros(0, 64), per_row=False)
    with pytest.raises(C.QmoeError, match="gradient"):
        D.quantize(torch.zeros(2, 64, requires_grad=True))
    rows = {"fmt": "nvfp4_rows", "w": torch.zeros(2, 32, dtype=torch.uint8), "sc": torch.zeros(2, 4, dtype=torch.uint8),
            "s": torch.ones(2), "N": 2, "K": 64}
    fp8 = {"fmt": "fp8", "w": torch.zeros(2, 64, dtype=torch.uint8), "s": torch.ones(1), "N": 2, "K": 64}
    with pytest.raises(C.QmoeError, match="scale per row"):
        D.gemv(rows, torch.zeros(64))
    with pytest.raises(C.QmoeError, match="NVFP4"):
        D.prepare(fp8)
    with pytest.raises(C.QmoeError, match="NVFP4"):
        D.gemm(fp8, rows)
    with pytest.raises(C.QmoeError, match="elements per"):
        D.gemm({**rows, "K": 128}, rows)
    with pytest.raises(C.QmoeError, match="32"):
        D.gemm({**rows, "K": 48}, {**rows, "K": 48})
    with pytest.raises(C.QmoeError, match="act"):
        D.gemm(rows, rows, act="gelu")
    with pytest.raises(C.QmoeError, match="act"):
        D.gemm(rows, rows, act="relu2", residual=torch.zeros(2, 2, dtype=torch.bfloat16))
    with pytest.raises(C.QmoeError, match="residual"):
        D.gemm(rows, rows, residual=torch.zeros(2, 3, dtype=torch.bfloat16))
    with pytest.raises(C.QmoeError, match="dtype"):
        D.gemm(rows, rows, dtype=torch.float64)


def test_an_operand_is_looked_at_in_every_call():
    """A dict whose tensors no longer belong together is refused, with its laid-out scales too: the kernels trust sizes."""
    import _qmoe_lib as C
    import dense_q as D
    q = {"fmt": "nvfp4", "w": torch.zeros(4, 32, dtype=torch.uint8), "sc": torch.zeros(4, 4, dtype=torch.uint8), "s": torch.ones(1),
         "sca": torch.zeros(512, dtype=torch.uint8), "N": 4, "K": 64}
    for bad, word in (({"w": q["w"][:3]}, "w must"), ({"w": torch.zeros(4, 64, dtype=torch.uint8)[:, ::2]}, "w must"),
                      ({"sc": q["sc"][:3]}, "sc must"), ({"s": torch.ones(2)}, "s must"), ({"sca": q["sca"][:256]}, "sca must"),
                      ({"sca": torch.zeros(512)}, "sca must"), ({"N": 129}, "w must")):
        with pytest.raises(C.QmoeError, match=word):
            D.gemm({**q, **bad}, q)
        with pytest.raises(C.QmoeError, match=word):
            D.gemm(q, {**q, **bad})


def test_dequant_alignment(lib):
    a = P(256)
    assert lib.dq_dequant_nvfp4(a, a, P(258), 1, 4, 64, 0, 4, a, 1, None) == 2
    assert lib.dq_dequant_nvfp4(a, a, a, 1, 4, 64, 0, 4, P(257), 1, None) == 2
    assert lib.dq_dequant_nvfp4(a, a, a, 1, 4, 64, 0, 4, P(258), 0, None) == 2


def test_linear_arguments(lib):
    a = P(256)
    need = lib.dq_linear_a4_workspace_bytes(5, 64)
    assert need == 5 * 32 + 512 + 32 + 5 * 4
    assert lib.dq_linear_a4_workspace_bytes(0, 64) == 0 and lib.dq_linear_a4_workspace_bytes(4, 48) == 0

    def call(w=a, x=a, dt=1, ldx=64, M=5, N=8, K=64, ep=0, res=None, y=a, ws=a, n=need):
        return lib.dq_linear_a4(w, a, a, a, 0, x, dt, ldx, M, N, K, ep, res, y, ws, n, None)

    assert call(w=None) == 5 and call(x=None) == 5 and call(y=None) == 5 and call(ws=None) == 5 and call(ep=2) == 5
    assert call(M=0) == 1 and call(N=0) == 1 and call(K=16) == 1 and call(ep=3) == 1 and call(ldx=63) == 1
    assert call(ws=P(264)) == 2 and call(n=need - 1) == 8 and call(dt=9) == 6
    if not torch.cuda.is_available():
        assert call() == 7 and call(M=4, ws=None, n=0) == 7    # few rows need no workspace


def test_prepare_looks_at_the_weight():
    import _qmoe_lib as C
    import dense_q as D
    q = {"fmt": "nvfp4", "w": torch.zeros(4, 32, dtype=torch.uint8), "sc": torch.zeros(4, 4, dtype=torch.uint8),
         "s": torch.ones(1), "N": 4, "K": 64}
    for bad in ({"w": torch.zeros(4, 31, dtype=torch.uint8)}, {"w": torch.zeros(4, 64, dtype=torch.uint8)[:, ::2]},
                {"sc": torch.zeros(4, 4)}, {"s": torch.ones(4)}, {"s": torch.ones(1, dtype=torch.float64)}, {"fmt": "nvfp4_rows"}, {}):
        with pytest.raises(C.QmoeError):
            D.prepare({**q, **bad})


def test_a_cpu_tensor_has_no_stream():
    import _qmoe_lib as C
    import dense_q as D
    q = {"fmt": "nvfp4", "w": torch.zeros(4, 32, dtype=torch.uint8), "sc": torch.zeros(4, 4, dtype=torch.uint8), "s": torch.ones(1), "N": 4, "K": 64}
    with pytest.raises(C.QmoeError, match="CUDA tensors"):
        D.gemv(q, torch.zeros(64))


def test_the_inverse_looks_at_its_tensors():
    """What is read has to be there: sizes, types and layout of every tensor, before any launch."""
    import _qmoe_lib as C
    import dense_q as D
    one = {"fmt": "nvfp4", "w": torch.zeros(4, 32, dtype=torch.uint8), "sc": torch.zeros(4, 4, dtype=torch.uint8), "s": torch.ones(1), "N": 4, "K": 64}
    rows = {**one, "fmt": "nvfp4_rows", "s": torch.ones(4)}
    out = torch.zeros(4, 64)
    for q, s in ((one, torch.ones(4)), (rows, torch.ones(1))):
        for bad, word in (({"w": q["w"][:3]}, "w must"), ({"w": torch.zeros(4, 64, dtype=torch.uint8)[:, ::2]}, "w must"), ({"w": torch.zeros(4, 32)}, "w must"),
                          ({"sc": q["sc"][:3]}, "sc must"), ({"sc": torch.zeros(4, 8, dtype=torch.uint8)[:, ::2]}, "sc must"), ({"s": s}, "s must"),
                          ({"s": q["s"].double()}, "s must"), ({"N": 5}, "w must"), ({"K": 128}, "w must"), ({"K": 8}, "multiple of 16"), ({}, "CUDA tensors")):
            with pytest.raises(C.QmoeError, match=word):
                D.dequant({**q, **bad})
            if q is rows:
                with pytest.raises(C.QmoeError, match=word):
                    D.dequant_rows({**q, **bad}, 0, 4, out)


def test_forward_mode_tangents_are_refused():
    """They are carried on under no_grad as well, so that a result without one would be silently wrong."""
    import _qmoe_lib as C
    import dense_q as D
    import torch.autograd.forward_ad as fwd
    rows = {"fmt": "nvfp4_rows", "w": torch.zeros(2, 32, dtype=torch.uint8), "sc": torch.zeros(2, 4, dtype=torch.uint8),
            "s": torch.ones(2), "N": 2, "K": 64}
    x = torch.zeros(2, 64)
    for grad in (True, False):
        with fwd.dual_level(), torch.set_grad_enabled(grad):
            dual, res = fwd.make_dual(x, torch.ones_like(x)), fwd.make_dual(torch.zeros(2, 2, dtype=torch.bfloat16), torch.ones(2, 2, dtype=torch.bfloat16))
            for bad in (lambda: D.quantize(dual), lambda: D.qlinear_a4(rows, dual), lambda: D.gemm(rows, rows, residual=res)):
                with pytest.raises(C.QmoeError, match="forward-mode"):
                    bad()


def test_few_rows_need_no_scale_atoms(lib):
    a = P(256)
    need = lib.dq_linear_a4_workspace_bytes(5, 64)

    def call(atoms, M):
        return lib.dq_linear_a4(a, a, atoms, a, 0, a, 1, 64, M, 8, 64, 0, None, a, a, need, None)

    assert call(None, 5) == 5 and call(None, 4) != 5
