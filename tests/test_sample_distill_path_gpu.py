"""The paths that use the operators on a model's distribution: continuations
sampled from one prompt (cngpt_cuda_generate_shared), a teacher's top logits
(cngpt_cuda_teacher_topk), the distillation step (cngpt_cuda_distill_step), and
the three of them in a row.

The reference values are the library's own gpt_forward logits of the full
sequences (held to the reference's CPU build elsewhere, normwise 1e-5) and the
definitions in 64 bits of test_distribution_ops_gpu.
"""
import ctypes as C

import numpy as np
import pytest
import torch

from cngpt_b200 import abi
from oracle import oracle
from tests.models import CudaModel, nwerr
from tests.test_distribution_ops_gpu import ref_distill, ref_sample

pytestmark = pytest.mark.gpu
HYPER = (0.9, 0.95, 1e-8, 0.1, 0.0)  # beta1, beta2, eps, wd, clip


@pytest.fixture()
def fast(lib):
    f = abi.FastCtx()
    lib.fast_init(C.byref(f))
    yield f
    lib.fast_free(C.byref(f))


def boosted(lib, L, H, Cm, V, block, seed):
    """A model whose logits spread over several units, as a trained one's do."""
    m = CudaModel(lib, L, H, Cm, V, block, seed)
    m.set_params(m.params() * np.float32(6.0))
    return m


def shared(lib, m, f, prompt, n, n_new, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    out = np.full(n * n_new, -9, np.int32)
    abi.check(lib, lib.cngpt_cuda_generate_shared(C.byref(m.m), C.byref(f), oracle.ptr(prompt), len(prompt), n, n_new,
                                                  temperature, top_k, top_p, min_p, u if isinstance(u, int) else oracle.ptr(u),
                                                  out.ctypes.data), "generate_shared")
    return out.reshape(n, n_new)


def check_draws(m, prompt, got, u, temperature, top_k, top_p, min_p):
    """Every token against the definition on the logits of the sequence so far.
    The decode path's logits differ from the full forward's by rounding (1e-5 of
    the largest), so a token also counts as right if the definition takes it for
    a number within 1e-3 of u; those are counted."""
    n, n_new = got.shape
    T = len(prompt)
    seq = np.concatenate([np.tile(prompt, (n, 1)), got], 1).astype(np.int32)
    S = T + n_new - 1
    flat = np.ascontiguousarray(seq[:, :S]).ravel()
    m.forward(flat, None, n, S)
    lg = m.logits(n, S)
    off = 0
    for q in range(n):
        for i in range(n_new):
            x, v = lg[q, T - 1 + i], float(u[i, q])
            draw = lambda w: ref_sample(x, temperature, top_k, top_p, min_p, w)[0]  # noqa: E731
            if got[q, i] == draw(v):
                continue
            off += 1
            assert got[q, i] in {draw(min(max(v + d, 0.0), 0.999999)) for d in np.linspace(-1e-3, 1e-3, 21)}, (q, i)
    assert off <= max(1, n * n_new // 50), off


@pytest.mark.parametrize("n,n_new", [(1, 1), (1, 9), (3, 2), (8, 3), (5, 12), (9, 7), (20, 10)])
@pytest.mark.parametrize("H,Cm,V,T", [(2, 128, 96, 11), (4, 32, 70, 1), (3, 192, 1001, 40)])
def test_generate_shared(lib, cuda, fast, n, n_new, H, Cm, V, T):
    m = boosted(lib, 2, H, Cm, V, 64, 5)
    prompt = oracle.lcg_tokens(T, V, seed=3)
    u = np.random.default_rng(n * n_new + T).random((n_new, n)).astype(np.float32)
    for kw in (dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0), dict(temperature=0.8, top_k=20, top_p=0.9, min_p=0.01)):
        got = shared(lib, m, fast, prompt, n, n_new, u, **kw)
        assert ((got >= 0) & (got < V)).all()
        check_draws(m, prompt, got, u, **kw)
        assert np.array_equal(got, shared(lib, m, fast, prompt, n, n_new, u, **kw))  # repeatable
    m.free()


def test_generate_shared_greedy_is_generate(lib, cuda, fast):
    m = boosted(lib, 2, 2, 128, 96, 64, 6)
    prompt = oracle.lcg_tokens(10, 96, seed=4)
    u = np.zeros((30, 4), np.float32)
    got = shared(lib, m, fast, prompt, 4, 30, u, temperature=0.0)
    g = abi.FastCtx()
    lib.fast_init(C.byref(g))
    want = np.zeros(30, np.int32)
    abi.check(lib, lib.cngpt_cuda_generate(C.byref(m.m), C.byref(g), oracle.ptr(prompt), 1, 10, 30, want.ctypes.data))
    lib.fast_free(C.byref(g))
    # the two decode paths' logits differ by rounding; these rows have no near-tie
    assert (got == want[None, :]).all()
    m.free()


def test_generate_shared_reuses_a_context(lib, cuda, fast):
    """Other numbers of sequences, lengths, prompts and models through one
    context give what a fresh context gives; device arrays work as host ones."""
    ms = [boosted(lib, 2, 2, 128, 96, 64, 7), boosted(lib, 3, 3, 192, 300, 64, 8)]
    rng = np.random.default_rng(1)
    for k, (n, T, n_new) in enumerate([(6, 9, 8), (6, 9, 8), (2, 30, 20), (12, 5, 4), (6, 20, 3), (12, 5, 9), (6, 9, 8)]):
        m = ms[k % 2]
        prompt = oracle.lcg_tokens(T, m.cfg.vocab_size, seed=k)
        u = rng.random((n_new, n)).astype(np.float32)
        a = shared(lib, m, fast, prompt, n, n_new, u, top_k=30)
        f2 = abi.FastCtx()
        lib.fast_init(C.byref(f2))
        du = torch.from_numpy(u).cuda()
        b = shared(lib, m, f2, prompt, n, n_new, du.data_ptr(), top_k=30)
        lib.fast_free(C.byref(f2))
        assert np.array_equal(a, b)
        # the greedy decode through the same context still is what it was
        out = np.zeros(5, np.int32)
        abi.check(lib, lib.cngpt_cuda_generate(C.byref(m.m), C.byref(fast), oracle.ptr(prompt), 1, T, 5, out.ctypes.data))
        lib.fast_init(C.byref(f2))
        out2 = np.zeros(5, np.int32)
        abi.check(lib, lib.cngpt_cuda_generate(C.byref(m.m), C.byref(f2), oracle.ptr(prompt), 1, T, 5, out2.ctypes.data))
        lib.fast_free(C.byref(f2))
        assert np.array_equal(out, out2)
    for m in ms:
        m.free()


def test_generate_shared_with_broken_weights_stays_in_bounds(lib, cuda, fast):
    m = CudaModel(lib, 1, 2, 128, 96, 64, 9)
    m.set_params(np.full(m.n, np.nan, np.float32))
    got = shared(lib, m, fast, oracle.lcg_tokens(5, 96, seed=1), 3, 6, np.full((6, 3), 0.5, np.float32))
    assert (got == -1).all()
    m.free()


def test_generate_shared_refuses_bad_arguments(lib, cuda, fast):
    m = CudaModel(lib, 1, 2, 64, 50, 16, 3)
    p, u, o = np.zeros(10, np.int32), np.zeros(100, np.float32), np.zeros(100, np.int32)
    call = lambda T, n, k, uu=u.ctypes.data: lib.cngpt_cuda_generate_shared(  # noqa: E731
        C.byref(m.m), C.byref(fast), p.ctypes.data, T, n, k, 1.0, 0, 1.0, 0.0, uu, o.ctypes.data)
    for bad in (call(10, 2, 8), call(0, 2, 2), call(4, 0, 2), call(4, 2, 0), call(4, 5000, 2), call(4, 2, 2, None)):
        assert bad == abi.ERR_ARG
    assert call(10, 2, 7) == abi.OK
    other = abi.GPT()
    assert lib.cngpt_cuda_generate_shared(C.byref(other), C.byref(fast), p.ctypes.data, 4, 2, 2, 1.0, 0, 1.0, 0.0,
                                          u.ctypes.data, o.ctypes.data) == abi.ERR_STATE
    lib.cngpt_cuda_clear_status()
    m.free()


def teacher_lists(lib, m, f, tok, B, T, k):
    v = torch.full((B * T, k), 7.0, device="cuda")
    i = torch.full((B * T, k), -7, dtype=torch.int32, device="cuda")
    abi.check(lib, lib.cngpt_cuda_teacher_topk(C.byref(m.m), C.byref(f), oracle.ptr(tok), B, T, k, v.data_ptr(), i.data_ptr()),
              "teacher_topk")
    abi.check(lib, lib.cngpt_cuda_check())
    return v, i


@pytest.mark.parametrize("L,B,T,V,k", [(2, 1, 1, 96, 5), (2, 3, 40, 96, 96), (0, 2, 7, 33, 4), (3, 5, 64, 1001, 64),
                                       (1, 20, 64, 4001, 10)])
def test_teacher_topk(lib, cuda, fast, L, B, T, V, k):
    m = boosted(lib, L, 2, 128, V, 64, 11)
    tok = oracle.lcg_tokens(B * T, V, seed=12)
    v, i = (t.cpu().numpy() for t in teacher_lists(lib, m, fast, tok, B, T, k))
    m.forward(tok, None, B, T)
    lg = m.logits(B, T).reshape(B * T, V)
    top = -np.sort(-lg, 1)[:, :k]
    tol = 1e-5 * np.abs(lg).max()  # the two forwards' logits differ by rounding
    assert np.abs(v - top).max() <= tol
    assert np.abs(np.take_along_axis(lg, i, 1) - v).max() <= tol
    assert (np.diff(v, axis=1) <= 0).all() and all(len(set(r)) == k for r in i.tolist())
    m.free()


def step(lib, m, tok, tgt, v, i, tau, alpha, B, T, lr=0.0):
    loss = C.c_float()
    k = 0 if v is None else v.shape[1]
    abi.check(lib, lib.cngpt_cuda_distill_step(C.byref(m.m), oracle.ptr(tok), None if tgt is None else oracle.ptr(tgt),
                                               None if v is None else v.data_ptr(), None if i is None else i.data_ptr(), k, tau,
                                               alpha, B, T, lr, *HYPER, C.byref(loss)), "distill_step")
    return loss.value, m.grads()


def hard_step(lib, m, tok, tgt, B, T, lr=0.0):
    loss = C.c_float()
    abi.check(lib, lib.cngpt_cuda_train_step(C.byref(m.m), oracle.ptr(tok), oracle.ptr(tgt), B, T, lr, *HYPER,
                                             C.byref(loss)), "train_step")
    return loss.value, m.grads()


def test_distill_step_without_a_teacher_is_the_training_step(lib, cuda):
    B, T, V = 3, 50, 1001
    m = CudaModel(lib, 2, 2, 128, V, 64, 13)
    tok, tgt = oracle.lcg_tokens(B * T, V, seed=1), oracle.lcg_tokens(B * T, V, seed=2)
    l0, g0 = hard_step(lib, m, tok, tgt, B, T)
    l1, g1 = step(lib, m, tok, tgt, None, None, 1.0, 0.0, B, T)
    assert abs(l0 - l1) <= 1e-6 * abs(l0) and nwerr(g1, g0) < 1e-5
    # a list of the target alone is a hard target too
    one = torch.from_numpy(tgt.reshape(-1, 1).copy()).cuda()
    l2, g2 = step(lib, m, tok, None, torch.zeros(B * T, 1, device="cuda"), one, 1.0, 1.0, B, T)
    assert abs(l0 - l2) <= 1e-6 * abs(l0) and nwerr(g2, g0) < 1e-5
    m.free()


@pytest.mark.parametrize("dropout", [0.0, 0.2])
def test_distill_step_mixes_targets_linearly(lib, cuda, dropout):
    """Two equal entries at temperature 1: the mean of the two hard gradients."""
    B, T, V = 2, 33, 515
    m = CudaModel(lib, 2, 2, 128, V, 64, 14, dropout=dropout)
    tok = oracle.lcg_tokens(B * T, V, seed=1)
    a = oracle.lcg_tokens(B * T, V, seed=5)
    b = ((a + 7) % V).astype(np.int32)

    def seeded(fn, *args):
        oracle.libc_rand_stream(99)  # the dropout masks
        return fn(*args)
    (la, ga), (lb, gb) = (seeded(hard_step, lib, m, tok, t, B, T) for t in (a, b))
    two = torch.from_numpy(np.stack([a, b], 1).copy()).cuda()
    l, g = seeded(step, lib, m, tok, None, torch.zeros(B * T, 2, device="cuda"), two, 1.0, 1.0, B, T)
    # the loss is the mean of the two less the list's entropy log 2
    assert abs(l - ((la + lb) / 2 - np.log(2.0))) <= 2e-6 * abs(la)
    assert nwerr(g, (ga.astype(np.float64) + gb) / 2) < 1e-5
    m.free()


def test_distill_step_refuses_bad_arguments(lib, cuda):
    m = CudaModel(lib, 1, 2, 64, 50, 16, 3)
    tok = np.zeros(8, np.int32)
    d = torch.zeros(8, 4, device="cuda")

    def call(tgt, v, k, tau, alpha):
        return lib.cngpt_cuda_distill_step(C.byref(m.m), tok.ctypes.data, tgt, v, d.data_ptr(), k, tau, alpha, 1, 8, 0.0, *HYPER,
                                           None)
    for bad in (call(None, d.data_ptr(), 4, 1.0, 0.5), call(None, None, 4, 1.0, 1.0), call(None, d.data_ptr(), 1025, 1.0, 1.0),
                call(None, d.data_ptr(), 4, 0.0, 1.0), call(None, d.data_ptr(), 4, 1.0, 1.5),
                call(None, tok.ctypes.data, 4, 1.0, 1.0)):
        assert bad == abi.ERR_ARG
    lib.cngpt_cuda_clear_status()
    m.free()


def test_sample_then_label_then_distil(lib, cuda, fast):
    """A teacher continues one prompt many times, its top logits on these
    sequences are recorded, and a smaller student takes a step on them: the
    loss and the logits' gradient are those of the definition on the two
    models' own logits, and the step moves the parameters."""
    V, T0, n, n_new, k, tau, alpha = 1001, 12, 6, 30, 16, 2.0, 0.7
    teacher, student = boosted(lib, 3, 4, 256, V, 64, 21), boosted(lib, 1, 2, 128, V, 64, 22)
    prompt = oracle.lcg_tokens(T0, V, seed=2)
    u = np.random.default_rng(3).random((n_new, n)).astype(np.float32)
    got = shared(lib, teacher, fast, prompt, n, n_new, u, temperature=0.9, top_p=0.95)
    seq = np.concatenate([np.tile(prompt, (n, 1)), got], 1).astype(np.int32)
    T = seq.shape[1] - 1
    tok, tgt = np.ascontiguousarray(seq[:, :-1]).ravel(), np.ascontiguousarray(seq[:, 1:]).ravel()
    v, i = teacher_lists(lib, teacher, fast, tok, n, T, k)
    student.forward(tok, None, n, T)
    x = student.logits(n, T).reshape(n * T, V)
    want = ref_distill(x, v.cpu().numpy(), i.cpu().numpy(), tgt, tau, alpha, 1.0 / (n * T))[0]
    before = student.params()
    loss, g = step(lib, student, tok, tgt, v, i, tau, alpha, n, T, lr=1e-3)
    assert abs(loss - want) <= 1e-5 * abs(want)
    assert np.isfinite(g).all() and np.abs(g).max() > 0
    after = student.params()
    assert np.isfinite(after).all() and not np.array_equal(before, after)
    # The gradient of the parameters against central differences along it. With
    # the steps h and h / 2 the second order's part of the difference's error is
    # taken off by extrapolation; h changes the loss by a two-thousandth, so what
    # is left of it is of the fourth order, and the losses, exact to about 1e-6 of
    # themselves, leave 4 / 3 * 1e-6 / 5e-4 = 0.3 %: one percent in all.
    student.set_params(before)
    size = float(np.linalg.norm(g))
    d = g.astype(np.float64) / size

    def difference(h):
        lp = []
        for s in (1, -1):
            student.set_params((before + s * h * d).astype(np.float32))
            lp.append(step(lib, student, tok, tgt, v, i, tau, alpha, n, T)[0])
        return (lp[0] - lp[1]) / (2 * h)
    h = 5e-4 * loss / size
    assert abs((4 * difference(h / 2) - difference(h)) / 3 - size) <= 1e-2 * size
    teacher.free()
    student.free()
