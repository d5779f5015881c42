"""CPU checks around the student ops: the plain forms that the GPU tests compare with, and what the entry points refuse before
anything reaches a device."""
import ctypes

import numpy as np
import pytest

from zigrad_b200 import abi
from zigrad_b200.device import USIZE, CudaDevice, DeviceSlice

from . import student


def rng(seed):
    return np.random.Generator(np.random.PCG64(seed))


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("twice", [False, True])
def test_gradient_of_the_plain_form_against_differences(tail, twice):
    g = rng(5)
    x, T, k = g.standard_normal((3, 11)) * 2, 1.7, 4
    index = np.stack([g.permutation(11)[:k] for _ in range(3)]).astype(np.uint64)
    if twice:
        index[0, 3] = index[0, 1]
    index[2, 2:] = 11  # a shorter list
    u = g.standard_normal((3, k)) * 2
    t_lse = np.array([3.0, 2.5, 4.0]) if tail else None
    _, grad, _ = student.distill(x, index, u, t_lse, None, T, 2.0)
    loss = lambda y: student.distill(y, index, u, t_lse, None, T, 2.0)[0].sum() / 2.0
    h = 1e-5
    for r in range(3):
        for j in range(11):
            e = np.zeros_like(x)
            e[r, j] = h
            # truncation h^2 f''' / 6 below 1e-10, rounding of the loss 1e-16 * 10 / h = 1e-10
            assert abs((loss(x + e) - loss(x - e)) / (2 * h) - grad[r, j]) <= 1e-9


def test_gradient_of_a_student_that_knows_nothing_but_the_list():
    """All else is -infinity and the teacher has half its mass there: no p_r, so r counts as 0 in the loss and in its gradient."""
    x, index, u, t_lse = np.array([[1.0, 0.5, -np.inf, -np.inf]]), np.array([[0, 1]], np.uint64), np.array([[1.0, 0.0]]), np.array([2.0])
    _, grad, part = student.distill(x, index, u, t_lse)
    assert 0.49 < 1 - part["mass"][0] < 0.5
    h = 1e-5
    for j in range(2):
        e = np.zeros_like(x)
        e[0, j] = h
        d = (student.distill(x + e, index, u, t_lse)[0] - student.distill(x - e, index, u, t_lse)[0])[0] / (2 * h)
        assert abs(d - grad[0, j]) <= 1e-9  # as above
    assert abs(grad.sum()) <= 1e-14  # a softmax does not change with a constant added to all of its logits


def test_divergence_is_zero_where_student_and_teacher_agree():
    x = rng(1).standard_normal((2, 20))
    v, i, l = student.top_logits(x, 6)
    row, grad, _ = student.distill(x, i, v, l)
    assert np.abs(row).max() <= 1e-14 and np.abs(grad).max() <= 1e-14


def test_verified_tokens_are_distributed_as_the_target():
    """Over all random numbers of a fine grid the first token's frequencies are the target's, whatever the draft's are."""
    C, N = 4, 64
    p, q = np.array([0.5, 0.125, 0.25, 0.125]), np.array([0.25, 0.5, 0.125, 0.125])
    count = np.zeros(C)
    for d in range(C):
        for i in range(N):
            for j in range(N):
                out, _ = student.verify(np.stack([p, p])[None], q[None, None], np.array([[d]]), None, np.array([[(i + 0.5) / N, (j + 0.5) / N]]))
                count[int(out[0, 0])] += q[d] / N / N
    np.testing.assert_allclose(count, p, atol=2.0 / N)


P = ctypes.c_void_p(1 << 20)  # never read: every call below is refused
S0 = abi.StreamWrapper(0)


def refused(code, call, *args):
    L = abi.lib()
    L.zg_clear_error()
    getattr(L, call)(*args)
    got, text = L.zg_last_error(), L.zg_last_error_message().decode()
    L.zg_clear_error()
    assert got == code and call in text, (got, text)


BAD, UNSUPPORTED = 2, 5


def top(**kw):
    d = dict(id=abi.SINGLE, x=P, rows=4, C=10, ld=0, k=3, T=1.0, v=P, i=P, lse=P)
    d.update(kw)
    return [d["id"], S0] + [d[n] for n in ("x", "rows", "C", "ld", "k", "T", "v", "i", "lse")]


@pytest.mark.parametrize("kw", [dict(rows=1 << 28), dict(C=0), dict(ld=9), dict(k=0), dict(k=11), dict(C=5000, k=1025), dict(T=0.0), dict(T=-1.0), dict(T=float("nan")),
                                dict(T=float("inf")), dict(T=1e-40), dict(C=1 << 31, k=1), dict(x=None), dict(v=None), dict(i=None),
                                dict(x=ctypes.c_void_p((1 << 20) + 2)), dict(i=ctypes.c_void_p((1 << 20) + 4)), dict(lse=ctypes.c_void_p((1 << 20) + 1))],
                         ids=str)
def test_top_logits_refuses(kw):
    refused(BAD, "zg_top_logits", *top(**kw))


def test_types_that_are_not_there():
    refused(UNSUPPORTED, "zg_top_logits", *top(id=abi.DOUBLE))
    refused(UNSUPPORTED, "zg_distill_ce", *ce(id=abi.DOUBLE))
    refused(UNSUPPORTED, "zg_distill_ce", *ce(t_id=abi.DOUBLE))
    refused(UNSUPPORTED, "zg_verify_drafts", *drafts(id=abi.DOUBLE))


def ce(**kw):
    d = dict(id=abi.SINGLE, t_id=abi.SINGLE, x=P, rows=4, C=10, ld=0, idx=P, u=P, lse=None, k=3, w=None, T=1.0, div=4.0, loss=P, row=P, grad=None, acc=0)
    d.update(kw)
    return [d["id"], d["t_id"], S0] + [d[n] for n in ("x", "rows", "C", "ld", "idx", "u", "lse", "k", "w", "T", "div", "loss", "row", "grad", "acc")]


@pytest.mark.parametrize("kw", [dict(rows=1 << 28), dict(C=0), dict(ld=9), dict(k=0), dict(k=1025), dict(T=0.0), dict(T=float("nan")), dict(div=0.0), dict(div=float("nan")),
                                dict(C=1 << 31), dict(x=None), dict(idx=None), dict(u=None), dict(loss=None), dict(row=None), dict(grad=P, acc=1),
                                dict(grad=ctypes.c_void_p((1 << 20) + 2)), dict(w=ctypes.c_void_p((1 << 20) + 2)), dict(idx=ctypes.c_void_p((1 << 20) + 4))],
                         ids=str)
def test_distill_ce_refuses(kw):
    refused(BAD, "zg_distill_ce", *ce(**kw))


def drafts(**kw):
    d = dict(id=abi.SINGLE, p=P, q=P, tok=P, n=None, u=P, batch=2, drafts=3, C=10, ldt=0, ldd=0, out=P, acc=P)
    d.update(kw)
    return [d["id"], S0] + [d[n] for n in ("p", "q", "tok", "n", "u", "batch", "drafts", "C", "ldt", "ldd", "out", "acc")]


@pytest.mark.parametrize("kw", [dict(C=0), dict(ldt=9), dict(ldd=9), dict(C=1 << 31), dict(drafts=1 << 31), dict(batch=1 << 31), dict(p=None), dict(tok=None), dict(u=None),
                                dict(out=None), dict(acc=None), dict(u=ctypes.c_void_p((1 << 20) + 2)), dict(tok=ctypes.c_void_p((1 << 20) + 4))], ids=str)
def test_verify_drafts_refuses(kw):
    refused(BAD, "zg_verify_drafts", *drafts(**kw))


def test_slices_are_looked_at():
    x = DeviceSlice(0, 40, abi.SINGLE)
    CudaDevice._fits("op", x=(x, 40, (abi.SINGLE, abi.BF16)), none=(None, 10, ()))
    with pytest.raises(ValueError):
        CudaDevice._fits("op", x=(x, 41, (abi.SINGLE,)))
    with pytest.raises(ValueError):  # of a negative size
        CudaDevice._fits("op", x=(x, -4, (abi.SINGLE,)))
    with pytest.raises(TypeError):
        CudaDevice._fits("op", x=(x, 4, (USIZE,)))


def test_the_cpp_host_side_has_the_three_ops(tmp_path):
    """Templates that nothing instantiates are not compiled: here they are."""
    import os
    import shutil
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "student_ops.cpp"
    ops = ("top_logits", "distill_ce", "verify_drafts")
    src.write_text('#include "zigrad_b200/host/cuda_device.hpp"\n' + "".join(
        "void run(zg::CudaDevice& d, const zg::opspec::%s<float>& p) { d.dispatch(p); }\n" % op for op in ops))
    done = subprocess.run([shutil.which("g++") or "g++", "-std=c++17", "-Wall", "-Werror", "-I", root, "-I", os.path.join(root, "include"),
                           "-fsyntax-only", str(src)], capture_output=True, text=True)
    assert done.returncode == 0, done.stderr
