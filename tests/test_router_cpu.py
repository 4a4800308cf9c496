"""What the router's operators refuse, checked without a GPU."""
import ctypes
import os

import pytest
import torch

P = ctypes.c_void_p


@pytest.fixture(scope="module")
def lib():
    import _qmoe_lib
    if not os.path.exists(_qmoe_lib.LIB_PATH):
        import qmoe_build
        qmoe_build.build()
    return _qmoe_lib.lib()


def test_route_arguments(lib):
    a = P(256)

    def call(x=a, dt=0, ld=512, bias=a, T=4, E=512, k=22, g=1, kg=1, score=0, ids=a, w=a, n=a):
        return lib.qmoe_route(x, dt, ld, bias, T, E, k, g, kg, 0, score, 5.0, ids, w, n, None)

    assert call(x=None) == 5 and call(ids=None) == 5 and call(w=None) == 5 and call(n=None) == 5
    assert call(T=0) == 1 and call(E=1025, ld=2000) == 1 and call(k=33) == 1 and call(k=0) == 1 and call(E=16, k=22) == 1
    assert call(ld=511) == 1 and call(g=3) == 1 and call(g=8, kg=9) == 1 and call(g=512, kg=4) == 1 and call(score=2) == 1
    assert call(score=1) == 1                              # a softmax router takes no bias
    assert call(dt=3) == 6 and call(x=P(257)) == 2
    if not torch.cuda.is_available():
        assert call() == 7 and call(bias=None, score=1) == 7 and call(g=8, kg=4) == 7

    def back(ids=a, dw=a, dl=a, T=4, k=22):
        return lib.qmoe_route_backward(a, 0, 512, T, 512, k, 0, 0, 5.0, ids, dw, dl, None)

    assert back(ids=None) == 5 and back(dw=None) == 5 and back(dl=None) == 5 and back(T=0) == 1 and back(k=33) == 1


def test_balance_arguments(lib):
    a = P(256)
    need = lib.qmoe_balance_workspace_bytes(100, 512)
    assert need > 0 and lib.qmoe_balance_workspace_bytes(0, 512) == 0 and lib.qmoe_balance_workspace_bytes(4, 1025) == 0

    def call(x=a, ids=a, T=100, E=512, k=22, loss=a, ws=a, n=need, score=0):
        return lib.qmoe_balance(x, 0, 512, ids, 1, None, T, E, k, score, 1.0, loss, a, a, ws, n, None)

    assert call(x=None) == 5 and call(ids=None) == 5 and call(loss=None) == 5 and call(ws=None) == 5
    assert call(T=0) == 1 and call(k=0) == 1 and call(score=3) == 1 and call(E=513) == 1
    assert call(ids=P(260)) == 2 and call(ws=P(257)) == 2 and call(n=need - 1) == 8
    assert lib.qmoe_balance_backward(a, 0, 512, None, 4, 512, 0, None, a, a, None) == 5
    assert lib.qmoe_balance_backward(a, 0, 500, None, 4, 512, 0, a, a, a, None) == 1
    if not torch.cuda.is_available():
        assert call() == 7


def test_misaligned_and_too_many(lib):
    a, b, c = P(256), P(258), P(260)

    def route(bias=None, ids=a, w=a, n=a, k=4, g=1, kg=1, score=0):
        return lib.qmoe_route(a, 0, 64, bias, 4, 64, k, g, kg, 0, score, 5.0, ids, w, n, None)

    assert route(bias=b) == 2 and route(ids=c) == 2 and route(w=b) == 2 and route(n=b) == 2
    assert route(k=17, g=8, kg=2, score=1) == 1            # a softmax leaves 16 experts in two of eight groups

    def back(ids=a, dw=a, dl=a, dt=0):
        return lib.qmoe_route_backward(a, dt, 64, 4, 64, 4, 0, 0, 5.0, ids, dw, dl, None)

    assert back(ids=c) == 2 and back(dw=b) == 2 and back(dl=b) == 2 and back(dl=P(257), dt=1) == 2

    def balance(T=100, k=22, loss=a, n=a, coef=a):
        return lib.qmoe_balance(a, 0, 64, a, 1, None, T, 64, k, 0, 1.0, loss, n, coef, a, 1 << 30, None)

    assert balance(loss=b) == 2 and balance(n=b) == 2 and balance(coef=b) == 2
    assert balance(T=1 << 30, k=2) == 1                    # 2^31 ids: a count may pass 32 bits
    assert lib.qmoe_balance_backward(a, 0, 64, None, 4, 64, 0, b, a, a, None) == 2
    assert lib.qmoe_balance_backward(a, 0, 64, None, 4, 64, 0, a, b, a, None) == 2
    assert lib.qmoe_balance_backward(a, 1, 64, None, 4, 64, 0, a, a, P(257), None) == 2
    if not torch.cuda.is_available():
        assert route() == 7 and route(k=16, g=8, kg=2, score=1) == 7 and back() == 7 and balance() == 7


def test_python_refusals():
    import _qmoe_lib as C
    import router as R
    x = torch.zeros(4, 64)
    ids = torch.zeros(4, 2, dtype=torch.int64)
    for bad in (lambda: R.route(x), lambda: R.route(torch.zeros(64)), lambda: R.route(torch.zeros(4, 1025)),
                lambda: R.route(torch.zeros(4, 64, dtype=torch.float64)), lambda: R.route(x, score="relu"),
                lambda: R.balance_loss(x, ids), lambda: R.balance_loss(x, ids, score="relu"),
                lambda: R.balance_loss(torch.zeros(4, 0), ids)):
        with pytest.raises(C.QmoeError):
            bad()
